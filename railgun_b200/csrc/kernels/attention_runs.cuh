// What the mma.sync kernels that read lists of cached entries for up to 16 queries share (bfloat16, head sizes 64, 128, 192 and 256, pages of
// 8 tokens or a larger power of two): a warp's ring of runs of 16 entries, what it does with a run, and how warps and the blocks of a
// cluster join what they have.
#pragma once
#include "common.cuh"
#include "mma.cuh"
#include "packed_f32.cuh"
#include "tcgen05.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;
using rgmma::mma_bf16;
using rgmma::pack_bf16;

#define PM_THREADS 128
#define PM_Q 16
// Runs of a warp's ring, and blocks an SM.  Head size 64: four and three (six and two, 12 % slower: 64 requests on 2,000 entries
// 70 against 63 us); 128: three and two (two and three are level, and 9 % slower for one request on 32,768).
// Brief: a warp has no more than two runs, and there are more blocks than 148 SMs hold at once, which then come and go: 128 requests' tokens on
// 100 entries 23.7 us (27.1 with the other), on 128 at head size 64 14.7 (17.1); with few blocks it is level or slower.
__host__ __device__ constexpr int pm_stages(int pieces, bool brief) {
    return brief ? (pieces == 1 ? 2 : 2) : (pieces == 1 ? 4 : (pieces == 3 ? 2 : 3));
}
__host__ __device__ constexpr int pm_blocks(int pieces, bool brief) {
    return brief ? (pieces == 1 ? 5 : 3) : (pieces == 1 ? 3 : (pieces == 2 ? 2 : 1));
}
static bool pm_brief(int d, long long entries, long long blocks) { return entries <= 128 && blocks > 148 * pm_blocks(d / 64, false); }
__host__ __device__ constexpr int pm_stage_bytes(int pieces) { return 16 * 64 * 2 * 2 * pieces; }
static_assert(4 * 4 * 16 * 64 <= 4 * pm_stages(1, true) * pm_stage_bytes(1), "the warps' results fit where the stages were");

// A run of 16 entries from entry e of its list on: one box, or where pages hold 8 tokens two.  One lane.
__device__ __forceinline__ void load_run(const CUtensorMap* map, int nkv, int page_size, uint32_t dst, uint32_t bar, int bytes, int box_shift, int page_a,
                                         int page_b, int kvh, int e) {
    mbar_expect_tx(bar, bytes);
    tma_load_4d_row(dst, map, bar, (page_a * 2 * nkv + kvh) * page_size + (e & (page_size - 1)));
    if (box_shift == 3) tma_load_4d_row(dst + bytes / 2, map, bar, (page_b * 2 * nkv + kvh) * page_size);
}
__device__ __forceinline__ void ldmatrix_x4_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

// A warp's 16 queries and what it has added up over the runs it has seen.
template <int PIECES>          // the head size in pieces of 64
struct MmaQueries {
    static constexpr int D = 64 * PIECES, KD = D / 16, ND = D / 8;
    uint32_t qf[KD][4];
    float o[ND][4], m0, m1, l0, l1;                                   // rows g and g + 8 of the tile
    uint32_t k_line, v_line, sw, k_c, v_c, piece;                     // where this lane's ldmatrix rows are in a stage
    int lane, g, tq, box_shift;

    // A stage is boxes of 1 << box_shift rows: K's 64-column pieces one after the other, then V's.
    __device__ __forceinline__ uint32_t line(int r) const {
        return (uint32_t)((((r >> box_shift) * 2 * PIECES) << box_shift) + (r & ((1 << box_shift) - 1))) * 128u;
    }
    __device__ __forceinline__ void init(int lane_, int box_shift_) {
        lane = lane_; g = lane >> 2; tq = lane & 3; box_shift = box_shift_;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.f;
        const int kr = (lane & 7) + (lane >> 4) * 8, vr = (lane & 7) + ((lane >> 3) & 1) * 8;   // K as the B operand, V transposed
        k_line = line(kr);
        v_line = line(vr) + (uint32_t)(PIECES << box_shift) * 128u;
        sw = (uint32_t)(lane & 7);
        k_c = (lane >> 3) & 1;
        v_c = lane >> 4;
        piece = (uint32_t)(128 << box_shift);
    }
    __device__ __forceinline__ void queries(const bf16* ra, const bf16* rb) {      // rows g and g + 8, null: zeros
#pragma unroll
        for (int k = 0; k < KD; ++k) {
            qf[k][0] = ra ? *reinterpret_cast<const uint32_t*>(ra + k * 16 + 2 * tq) : 0u;
            qf[k][1] = rb ? *reinterpret_cast<const uint32_t*>(rb + k * 16 + 2 * tq) : 0u;
            qf[k][2] = ra ? *reinterpret_cast<const uint32_t*>(ra + k * 16 + 8 + 2 * tq) : 0u;
            qf[k][3] = rb ? *reinterpret_cast<const uint32_t*>(rb + k * 16 + 8 + 2 * tq) : 0u;
        }
    }
    // The run in stage `st`, of which n entries are looked at (16 or more: all).  keep(v): the scores of row g, entries
    // 2 tq + {0, 1, 8, 9}, then those of row g + 8.
    template <typename Keep>
    __device__ __forceinline__ void step(uint32_t st, int n, float scale_log2, Keep keep) {
        if (n < 16) {
            // rows of V behind the last entry are what an earlier request left: 0 times an infinity is no number
            for (int j = lane; j < (16 - n) * 8 * PIECES; j += 32) {
                const int r = n + j / (8 * PIECES), c = j % (8 * PIECES);
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                             ::"r"(st + line(r) + (uint32_t)(PIECES << box_shift) * 128u + (c >> 3) * piece + (c & 7) * 16), "r"(0) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the stage's next box comes after these
            __syncwarp();
        }
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KD; ++k) {
            uint32_t b[4];
            ldmatrix_x4_at(b, st + k_line + (k >> 2) * piece + ((((k & 3) * 2 + k_c) ^ sw) << 4));
            mma_bf16(s0, qf[k], b[0], b[1]);
            mma_bf16(s1, qf[k], b[2], b[3]);
        }
        float v[8] = {s0[0], s0[1], s1[0], s1[1], s0[2], s0[3], s1[2], s1[3]};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] *= scale_log2;
            if (n < 16 && 2 * tq + (j & 1) + ((j & 2) << 2) >= n) v[j] = -INFINITY;
        }
        keep(v);
        float x0 = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), x1 = fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float r0 = n0 == -INFINITY ? 0.f : n0, r1 = n1 == -INFINITY ? 0.f : n1;
        if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {          // some row's maximum moved
            const float f0 = ex2(m0 - r0), f1 = ex2(m1 - r1);
            l0 *= f0; l1 *= f1;
#pragma unroll
            for (int j = 0; j < ND; ++j) { o[j][0] *= f0; o[j][1] *= f0; o[j][2] *= f1; o[j][3] *= f1; }
            m0 = n0; m1 = n1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] = ex2(v[j] - r0); v[j + 4] = ex2(v[j + 4] - r1); }
        l0 += (v[0] + v[1]) + (v[2] + v[3]);                          // this thread's entries; added up at the end
        l1 += (v[4] + v[5]) + (v[6] + v[7]);
        // weights to bfloat16, up to 2^-8 of each, for the second product (the sums above are of the weights before that rounding)
        const uint32_t p[4] = {pack_bf16(v[0], v[1]), pack_bf16(v[4], v[5]), pack_bf16(v[2], v[3]), pack_bf16(v[6], v[7])};
#pragma unroll
        for (int k = 0; k < KD; ++k) {                                // 16 columns at a time
            uint32_t b[4];
            ldmatrix_x4_trans_at(b, st + v_line + (k >> 2) * piece + ((((k & 3) * 2 + v_c) ^ sw) << 4));
            mma_bf16(o[2 * k], p, b[0], b[1]);
            mma_bf16(o[2 * k + 1], p, b[2], b[3]);
        }
        __syncwarp();                                                 // every lane has read the stage
    }
    __device__ __forceinline__ void sums() {                         // of the weights, over the four lanes of a row
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    }
    // What the warp has, to shared memory: co [16][D], ml [16][2].
    __device__ __forceinline__ void leave(float* co, float (*ml)[2]) {
        sums();
#pragma unroll
        for (int j = 0; j < ND; ++j) {
            *reinterpret_cast<float2*>(co + g * D + j * 8 + 2 * tq) = make_float2(o[j][0], o[j][1]);
            *reinterpret_cast<float2*>(co + (g + 8) * D + j * 8 + 2 * tq) = make_float2(o[j][2], o[j][3]);
        }
        if (tq == 0) { ml[g][0] = m0; ml[g][1] = l0; ml[g + 8][0] = m1; ml[g + 8][1] = l1; }
    }
};
// The four warps' results for row r, columns c .. c + 3: unnormalised sum, M and L.
template <int D>
__device__ __forceinline__ float4 join_warps(const float* all, const float (*ml)[PM_Q][2], int r, int c, float& M, float& L) {
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, ml[w][r][0]);
    const float ref = M == -INFINITY ? 0.f : M;
    float4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = ex2(ml[w][r][0] - ref);
        const float4 x = *reinterpret_cast<const float4*>(all + (w * PM_Q + r) * D + c);
        L += f * ml[w][r][1];
        sum.x += f * x.x; sum.y += f * x.y; sum.z += f * x.z; sum.w += f * x.w;
    }
    return sum;
}

// Query r's M and 1 / L (0 where no entry is seen; no number where a score is none) from what the blocks of a cluster have
// ([queries][2] each).
__device__ __forceinline__ void join_cluster_ml(cg::cluster_group& cluster, float* ml, int r, float& M, float& inv) {
    const int C = cluster.num_blocks();
    float m = -INFINITY, L = 0.f;
    for (int k = 0; k < C; ++k) m = fmaxf(m, cluster.map_shared_rank(ml, k)[r * 2]);
    M = m == -INFINITY ? 0.f : m;
    for (int k = 0; k < C; ++k) {
        const float* from = cluster.map_shared_rank(ml, k) + r * 2;
        L += exp2f(from[0] - M) * from[1];
    }
    inv = L == 0.f ? 0.f : 1.f / L;
}

// The cache as the mma kernel reads it: 64 columns, rows, pieces of 64 columns, K and V; a box of `rows` rows.
static int make_kv_map(CUtensorMap* map, const void* kv, int num_pages, int nkv, int page_size, int d, int rows) {
    RgEncodeTiledFn fn = rg_encode_fn();
    if (!fn) return RG_ERR_UNSUPPORTED;
    cuuint64_t dims[4] = {64, (cuuint64_t)num_pages * 2 * nkv * page_size, (cuuint64_t)(d / 64), 2};
    cuuint64_t strides[3] = {(cuuint64_t)d * 2, 128, (cuuint64_t)nkv * page_size * d * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)rows, (cuuint32_t)(d / 64), 2}, estr[4] = {1, 1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(kv), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 20000 + (int)r;
}
