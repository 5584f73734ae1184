// Trees of few nodes, or behind short contexts, in one launch: a cluster takes an item (a request, a kv head and up to 16 queries, rows x
// heads) and cuts its entries among its blocks, which join through each other's shared memory and leave the output (bfloat16, head
// sizes 64, 128, 192 and 256, mma.sync; attention_runs.cuh has what a warp does).  Entries are read again for every 16 queries, out of L2;
// what is saved is the plan, the second launch and the parts' trip through memory.  What bounds it is the launch and three trips to
// memory, for the request, the table and the entries: one request of 16 nodes, 32 heads on 8 of 64, on 1,024 entries takes 8.7 us (12.7 in
// stretches; 2 MB are 0.35 us of a copy), 8 chains of 5 with 24 heads on 8 of 128 on up to 2,000 entries 16.6 (24; 50 MB are 7.6).
#pragma once
#include "attention_runs.cuh"
#include "attention_tree.cuh"

// Which of the 16 entries from e on row t sees: those before start, and the nodes that its mask has.
__device__ __forceinline__ uint32_t tree_seen16(const TreeArgs& a, int t, int node) {
    const int first = max(node, 0), word = first >> 5;
    const int* mask = a.masks + (size_t)t * a.words;
    const uint32_t m0 = word < a.words ? (uint32_t)mask[word] : 0u, m1 = word + 1 < a.words ? (uint32_t)mask[word + 1] : 0u;
    const uint32_t bits = __funnelshift_r(m0, m1, first & 31);
    return node >= 0 ? bits : bits << -node | ((1u << -node) - 1);     // node > -16
}

template <int PIECES, bool BRIEF>
__global__ void __launch_bounds__(PM_THREADS, pm_blocks(PIECES, BRIEF))
tree_rows_kernel(const __grid_constant__ CUtensorMap kv_map, const TreeArgs a, bf16* __restrict__ out, int out_ld, int q_blocks) {
    constexpr int D = 64 * PIECES, STAGES = pm_stages(PIECES, BRIEF), STAGE = pm_stage_bytes(PIECES);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[4 * STAGES];
    __shared__ float ml[4][PM_Q][2], fin_ml[PM_Q][2], row_ml[PM_Q][2];
    __shared__ int abort_flag;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t first_stage = (smem_addr(smem_raw) + 1023u) & ~1023u, base = first_stage + (uint32_t)(warp * STAGES * STAGE);
    const uint32_t bar0 = smem_addr(bars) + (uint32_t)(8 * STAGES * warp);
    float* all = reinterpret_cast<float*>(smem_raw + (first_stage - smem_addr(smem_raw)));   // [4][16][D], then the block's [16][D]
    float* fin = all + 4 * PM_Q * D;
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        fence_barrier_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    TreeWalk item;
    if (!tree_item(a, blockIdx.x / C, q_blocks, item)) return;        // all blocks of the cluster
    const TreeRequest& x = item.x;
    const int group = a.nh / a.nkv, kvh = item.kvh(), q0 = item.block() * PM_Q, nq = min(PM_Q, x.rows * group - q0);
    const int total = (x.entries + 15) >> 4, per = (total + C - 1) / C, first = min(total, rank * per), last = min(total, first + per);
    const int n_runs = last - first, mine = n_runs > warp ? (n_runs - warp + 3) >> 2 : 0;
    const int* table = a.block_table + (size_t)item.r * a.max_blocks;
    const int box_shift = a.page_shift < 4 ? 3 : 4;
    int page_a = 0, page_b = 0;
    auto page_at = [&](int e) -> int {
        int page = table[e >> a.page_shift];
        if ((unsigned)page >= (unsigned)a.pages) { atomicCAS(a.err, 0, RG_BAD_PAGE); page = 0; }
        return page;
    };
    auto entry_of = [&](int i) -> int { return (first + warp + 4 * i) * 16; };
    auto issue = [&](int i) {                                         // the whole warp: run i of this warp
        if ((i & 31) == 0) {
            const int e = entry_of(i + lane);
            const bool there = i + lane < mine;
            page_a = there ? page_at(e) : 0;
            if (box_shift == 3) page_b = there && e + 8 < x.entries ? page_at(e + 8) : page_a;       // no such entry: any page
        }
        const int pa = __shfl_sync(0xffffffffu, page_a, i & 31), pb = __shfl_sync(0xffffffffu, page_b, i & 31);
        if (lane == 0) load_run(&kv_map, a.nkv, a.page_size, base + (i % STAGES) * STAGE, bar0 + 8 * (i % STAGES), STAGE, box_shift, pa, pb, kvh, entry_of(i));
        __syncwarp();
    };
    for (int i = 0; i < min(STAGES, mine); ++i) issue(i);
    MmaQueries<PIECES> w;
    w.init(lane, box_shift);
    const bool has_a = w.g < nq, has_b = w.g + 8 < nq;
    const int qa = q0 + min(w.g, nq - 1), qb = q0 + min(w.g + 8, nq - 1), ta = x.row0 + qa / group, tb = x.row0 + qb / group;
    w.queries(has_a ? (const bf16*)a.q + (size_t)ta * a.q_stride + (size_t)(kvh * group + qa % group) * D : nullptr,
              has_b ? (const bf16*)a.q + (size_t)tb * a.q_stride + (size_t)(kvh * group + qb % group) * D : nullptr);
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
        const int s = i % STAGES, e = entry_of(i), node = e - x.start;
        uint32_t seen_a = 0xffffu, seen_b = 0xffffu;
        if (node > -16) { seen_a = tree_seen16(a, ta, node); seen_b = tree_seen16(a, tb, node); }
        ok = mbar_wait_all(bar0 + 8 * s, (i / STAGES) & 1, a.err, 62, &abort_flag);
        if (!ok) break;
        w.step(base + s * STAGE, x.entries - e, a.scale_log2, [&](float (&v)[8]) {
            if (node > -16) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!((j < 4 ? seen_a : seen_b) >> (2 * w.tq + (j & 1) + ((j & 2) << 2)) & 1)) v[j] = -INFINITY;
            }
        });
        if (i + STAGES < mine) issue(i + STAGES);
    }
    if (!ok || abort_flag)                                            // give copies in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
    w.leave(all + warp * PM_Q * D, ml[warp]);
    __syncthreads();
    for (int idx = threadIdx.x; idx < nq * (D / 4); idx += PM_THREADS) {
        const int r = idx / (D / 4), c = idx % (D / 4) * 4;
        float M, L;
        *reinterpret_cast<float4*>(fin + r * D + c) = join_warps<D>(all, ml, r, c, M, L);
        if (c == 0) { fin_ml[r][0] = M; fin_ml[r][1] = L; }
    }
    cluster.sync();                                                   // every block's result is in place
    if (threadIdx.x < nq) join_cluster_ml(cluster, &fin_ml[0][0], threadIdx.x, row_ml[threadIdx.x][0], row_ml[threadIdx.x][1]);
    __syncthreads();
    // a warp has whole queries, so that it can work out again what is no number
    for (int r = rank * 4 + warp; r < nq; r += C * 4) {
        const int t = x.row0 + (q0 + r) / group, h = kvh * group + (q0 + r) % group;
        bf16* to = out + (size_t)t * out_ld + (size_t)h * D;
        bool odd = false;
        for (int c = lane * 4; c < D; c += 128) {
            float4 sum = {0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < C; ++k) {
                const float f = ex2(cluster.map_shared_rank(&fin_ml[0][0], k)[r * 2] - row_ml[r][0]) * row_ml[r][1];
                const float4 y = *reinterpret_cast<const float4*>(cluster.map_shared_rank(fin, k) + r * D + c);
                sum.x += f * y.x; sum.y += f * y.y; sum.z += f * y.z; sum.w += f * y.w;
            }
            odd |= !(isfinite(sum.x) && isfinite(sum.y) && isfinite(sum.z) && isfinite(sum.w));
            to[c] = __float2bfloat16_rn(sum.x); to[c + 1] = __float2bfloat16_rn(sum.y);
            to[c + 2] = __float2bfloat16_rn(sum.z); to[c + 3] = __float2bfloat16_rn(sum.w);
        }
        if (__any_sync(0xffffffffu, odd)) row_by_formula<bf16>(a, x, item.r, t, h, to, 0, D);
    }
    cluster.sync();                                                   // nobody leaves while its results are being read
}

// bfloat16, head sizes in pieces of 64, pages of a power of two from 8 on, rows of q on 4-byte boundaries, and addresses that fit the map's
// coordinates.
static bool tree_rows_ok(const TreeArgs& a, int dtype) {
    return dtype == RG_DTYPE_BF16 && a.d % 64 == 0 && a.page_shift >= 3 && a.q_stride % 2 == 0 && ((uintptr_t)a.q & 3) == 0 &&
           ((uintptr_t)a.kv & 15) == 0 && a.max_blocks > 0 && (long long)a.pages * 2 * a.nkv * a.page_size < 0x7fffffffll;
}

static int launch_tree_rows(const TreeArgs& a, bf16* out, int out_ld, int cluster, int q_blocks, cudaStream_t s) {
    CUtensorMap map;
    int e = make_kv_map(&map, a.kv, a.pages, a.nkv, a.page_size, a.d, a.page_size < 16 ? a.page_size : 16);
    if (e) return e;
    const long long blocks = (long long)a.R * a.nkv * q_blocks * cluster;
#define RG_TR(P, B) { constexpr int smem = 4 * pm_stages(P, B) * pm_stage_bytes(P) + 1024; \
    static_assert(5 * PM_Q * 64 * P * 4 <= 4 * pm_stages(P, B) * pm_stage_bytes(P), "the warps' and the block's results fit where the stages were"); \
    RG_ALLOW_SMEM((tree_rows_kernel<P, B>), smem) \
    return rg_launch(tree_rows_kernel<P, B>, dim3((unsigned)blocks), dim3(PM_THREADS), smem, s, cluster, map, a, out, out_ld, q_blocks); }
    const bool brief = pm_brief(a.d, (a.limit + cluster - 1) / cluster, blocks);
    if (a.d == 64) { if (brief) RG_TR(1, true) else RG_TR(1, false) }
    if (a.d == 128) { if (brief) RG_TR(2, true) else RG_TR(2, false) }
    if (a.d == 192) RG_TR(3, false)
    RG_TR(4, false)
#undef RG_TR
}
