// Trees of drafted tokens on the 5th-generation tensor cores (bfloat16, head sizes 64 and 128): the stretches that
// attention_tree.cuh describes.
//
// A block is one to an SM and stays; it has two sides of 128 queries (rows x heads of a kv head), each with its own softmax
// threads, accumulator and issuing warp.  Where a request brings up to 128 queries a kv head, the sides are two workers with a stretch
// each, so that two chains of scores, exponentials and products are under way on the SM; where it may bring more, the block
// is one worker, and K and V are fetched once for 256 queries.  K and V tiles of 128 entries (TMA through the request's table,
// one box a page and 64 columns, 128-byte swizzle) come through two rings that both sides share, and go on from one item
// to the next: while a side leaves one item's part and begins another's, tiles keep coming and the other side keeps computing.
// Per side and 64 entries j of an item:
//   S(j) = Q K^T         tcgen05.mma, M 128 x N 64 x K head size, into one of two buffers of 64 TMEM columns
//   softmax              128 threads, one query each; the reference maximum is raised only when the 64 weights sum to more than 2^8
//   O += P(j) V          tcgen05.mma, M 128 x N head size x K 64: P as bfloat16 in TMEM over the scores it was made from
// S(j + 2) is issued behind O += P(j) V, which reads the buffer that it goes to, so S(j + 1) is there when the threads are done
// with j.  Only passes that hold nodes of the tree, or the end of the list, look at masks: 64 bits a query.
//
// What bounds it, 32 heads on 8 of 128.  Few queries: the cache.  64 requests of 16 nodes behind up to 4,096 entries, 817 MB, take 134 us and 13 to
// join, 93 % of what a copy reaches; called on and on, the power limit takes the clock to 1.5 GHz and a call to 163 to 177.  Many: 128 nodes of
// one request on 65,536 entries take 132 us and 10 to join, 137 GFLOP, 83 us at the rate of a large product.  A pass of both sides takes
// 2,090 cycles there.  Alone its products take 1,300 (N 64 is bound by what it fetches from shared memory) and its exponentials 1,080, or 1,180
// where nothing but products runs beside them.  In the kernel a softmax warp spends 1,300 of the 2,090 on exponentials, 200 on storing weights and
// the rest on its loop and on waiting for the next scores: the sides fall into step, and neither covers the other's waits.  Slower, in us for these
// two, 149 and 148 then: an issuing warp for a side's even and one for its odd passes 153 and 155, the next scores loaded beside the store of
// the weights 154 and 158, passes of 128 entries and one issuing warp for both sides 161 and 171, two threads a query 167 and 152.
//
// Rounding: P to bfloat16 (up to 2^-8 of each weight; the sum of weights is of the unrounded ones), all sums in 32-bit.
#pragma once
#include "attention_tree.cuh"
#include "packed_f32.cuh"
#include "tcgen05.cuh"
#include <type_traits>

#define TT_SIDE 128                // queries of a side
#define TT_BN 64                   // entries of a softmax pass
#define TT_STAGE 128               // entries of a K or V stage: a tile
#define TT_THREADS 384             // warps 0-3, 4-7: softmax of side 0, 1; 8, 10: TMA of K, of V; 9, 11: MMA issue (and TMA of Q) of side 0, 1
#define TT_BARRIERS 384            // bytes
// Places in front of an item's tiles.  With 0, 2 and 3 of them: 4 requests of 64 nodes on 8,192 entries 59.0, 55.1 and 54.5 us, 64 of 16 behind up to
// 4,096 147.9, 146.2 and 148.1, 128 of 16 behind up to 500 74.4, 72.1 and 72.8, 128 nodes on 65,536 145.1, 141.8 and 141.8.
#define TT_BEGIN 2
__host__ __device__ constexpr int tt_k_stages(int pieces) { return pieces == 1 ? 5 : 3; }
__host__ __device__ constexpr int tt_v_stages(int pieces) { return pieces == 1 ? 4 : 2; }
__host__ __device__ constexpr int tt_smem(int pieces) {
    return (2 + tt_k_stages(pieces) + tt_v_stages(pieces)) * TT_SIDE * 128 * pieces + TT_BARRIERS + 1024;
}

__device__ __forceinline__ void tt_store8(float* p, const uint32_t (&v)[32], int i) {      // 32 bytes: a whole sector of the row
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]),
                 "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7]) : "memory");
}

// mbar_wait_all for three barriers at once.
__device__ __forceinline__ bool wait_all_of(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2, int* err, int code,
                                            volatile int* abort_flag) {
    for (uint32_t i = 0; i < RG_SPIN_LIMIT; ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p, q, r;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n\t"
                     "and.pred p, p, q;\n\t"
                     "and.pred p, p, r;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(b0), "r"(p0), "r"(b1), "r"(p1), "r"(b2), "r"(p2) : "memory");
        if (__all_sync(0xffffffffu, ok)) return true;
        if ((i & 1023u) == 1023u && __any_sync(0xffffffffu, *abort_flag)) return false;
    }
    atomicCAS(err, 0, code);
    *abort_flag = 1;
    return false;
}

// Which of the 64 entries from e on row t sees (n of them are there; n >= 1): those before start, and the nodes that its mask has.
__device__ __forceinline__ uint64_t tree_seen(const TreeArgs& a, int t, int start, int e, int n) {
    uint64_t seen = ~0ull;
    const int node = e - start;                                       // of the first entry; negative: before the tree
    if (node > -TT_BN) {
        const int first = max(node, 0), word = first >> 5, shift = first & 31;
        const int* mask = a.masks + (size_t)t * a.words;
        uint32_t m[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) m[i] = word + i < a.words ? (uint32_t)mask[word + i] : 0u;
        const uint64_t bits = (uint64_t)__funnelshift_r(m[0], m[1], shift) | (uint64_t)__funnelshift_r(m[1], m[2], shift) << 32;
        seen = node >= 0 ? bits : bits << -node | ((1ull << -node) - 1);
    }
    return n < TT_BN ? seen & ((1ull << n) - 1) : seen;
}

// q_map: 64 columns x heads x rows, a box of 64 x group x tile_rows (tile_rows rows fill a side, or are all there may be); kv_map: the
// cache as rows of the head size, a box of min(page, 128) rows x 64 columns.  both: the sides share a stretch.
template <int PIECES>
__global__ void __launch_bounds__(TT_THREADS, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const TreeArgs a, int tile_rows, int both) {
    extern __shared__ unsigned char smem_raw[];
    constexpr int D = 64 * PIECES, NK = tt_k_stages(PIECES), NV = tt_v_stages(PIECES);
    constexpr uint32_t PIECE = TT_STAGE * 128, TILE = PIECE * PIECES, SUB = TT_BN * 128;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sQ = base, sK0 = sQ + 2 * TILE, sV0 = sK0 + NK * TILE, bars = sV0 + NV * TILE;
    // A stage is full on the barrier of the side whose tile it holds (side 0's, where the tile is both sides').  A wait goes by the parity of
    // a phase, so that who waits has to have seen all phases before: of barriers that both sides' tiles came through in turn, a side would
    // see every second one, and take its tile for loaded while the other side's before it was still on its way.
    const uint32_t q_full0 = bars, k_full0 = bars + 16, k_empty0 = k_full0 + 16 * NK, v_full0 = k_empty0 + 8 * NK, v_empty0 = v_full0 + 16 * NV,
                   s_full0 = v_empty0 + 8 * NV, p_full0 = s_full0 + 32, p_free0 = p_full0 + 32;    // per side and half stage
    static_assert(16 + 24 * (NK + NV) + 96 <= TT_BARRIERS, "the barriers' place");
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ TreeStart st;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.nh / a.nkv;
    int* const err = a.err;
    if (threadIdx.x == 0) {
        const uint32_t users = both ? 2 : 1;
        abort_flag = 0;
        mbar_init(q_full0, 1);
        mbar_init(q_full0 + 8, 1);
        for (int s = 0; s < 2 * NK; ++s) mbar_init(k_full0 + 8 * s, 1);
        for (int s = 0; s < 2 * NV; ++s) mbar_init(v_full0 + 8 * s, 1);
        for (int s = 0; s < NK; ++s) mbar_init(k_empty0 + 8 * s, users);
        for (int s = 0; s < NV; ++s) mbar_init(v_empty0 + 8 * s, users);
        for (int b = 0; b < 4; ++b) { mbar_init(s_full0 + 8 * b, 1); mbar_init(p_full0 + 8 * b, TT_SIDE); mbar_init(p_free0 + 8 * b, 1); }
        fence_barrier_init();
    }
    if (threadIdx.x == 32) {
        tma_prefetch_map(&q_map);
        tma_prefetch_map(&kv_map);
    }
    pdl_wait();                                                       // tables, lengths and queries may come from the kernel before
    pdl_trigger();
    // side s's worker: the second sides' stretches come behind all first sides', so that little work is one stretch an SM
    auto worker_of = [&](int s) -> int { return blockIdx.x + (both ? 0 : s * (int)gridDim.x); };
    if (warp == 11) tmem_alloc(&tmem_base_slot, 512u);                // (all kernels before are over: nobody who has some waits for this block)
    tree_plan<TT_THREADS>(a, blockIdx.x, both ? 1 : 2, gridDim.x, st);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int n_t0 = st.tiles(0), n_t1 = both ? 0 : st.tiles(1);      // n_t1: of its own stretch
    if (n_t0 + n_t1 == 0) {
        if (warp == 11) tmem_free(tmem_base_slot, 512u);
        return;
    }
    // A stage of the stream belongs to both sides, or in turn to either while both have some, then to who has more
    const int n_stages = n_t0 + n_t1, n_turns = min(n_t0, n_t1);
    auto stages_on = [&](int s, int t) -> int {                       // from side s's tile t to its next
        return both || t >= n_turns ? 1 : t + 1 < n_turns ? 2 : 2 - s;
    };
    // side s: scores and weights in columns [256 s, 256 s + 128), O in [256 s + 128, 256 s + 128 + D)
    const uint32_t tmem = tmem_base_slot;

    if (warp == 8 || warp == 10) {
        // ---- producers of K and of V.  A stage is 128 / box_rows boxes for each 64 columns; lane l has box l % boxes of piece l / boxes.
        const int box_rows = min(a.page_size, TT_STAGE), boxes = TT_STAGE / box_rows, box = lane % boxes, piece = lane / boxes;
        const bool mine = piece < PIECES;
        TreeWalk w0, w1;
        if (n_t0) w0.at(a, st, 0);
        if (n_t1) w1.at(a, st, 1);
        int left0 = n_t0, left1 = n_t1;
        const int kv = warp == 10 ? 1 : 0, n = kv ? NV : NK;
        auto row_of = [&](TreeWalk& w, int& left) -> int {            // the cache's row of this lane's box; one tile on
            const int e = w.tile * TT_STAGE + box * box_rows;
            int page = a.block_table[(size_t)w.r * a.max_blocks + (e < w.x.entries ? e >> a.page_shift : 0)];   // behind the end: any page
            if ((unsigned)page >= (unsigned)a.pages) { atomicCAS(err, 0, RG_BAD_PAGE); page = 0; }
            const int row = ((page * 2 + kv) * a.nkv + w.kvh()) * a.page_size + (e & (a.page_size - 1));
            w.next(a, --left > 0);
            return row;
        };
        auto side_of = [&](int b) -> int { return b < 2 * n_turns ? b & 1 : n_t1 > n_t0; };
        auto look_up = [&](int b) -> int {                            // of stage b, one after the other
            if (b >= n_stages) return 0;
            return side_of(b) ? row_of(w1, left1) : row_of(w0, left0);
        };
        int row_next = look_up(0);
        bool ok = true;
        for (int b = 0; b < n_stages && ok; ++b) {
            const int row = row_next;
            row_next = look_up(b + 1);
            const int stage = b % n, u = b / n;
            const uint32_t full = (kv ? v_full0 : k_full0) + 8 * (stage + n * side_of(b)), empty = (kv ? v_empty0 : k_empty0) + 8 * stage;
            if (u > 0) ok = mbar_wait_all(empty, (u & 1) ^ 1, err, 71 + kv, &abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(full, TILE);
            __syncwarp();
            if (mine) tma_load_2d((kv ? sV0 : sK0) + stage * TILE + piece * PIECE + box * box_rows * 128, &kv_map, full, 64 * piece, row);
        }
    } else if (warp == 9 || warp == 11) {
        // ---- MMA issue of one side.  The whole warp walks the loop and waits; one elected lane issues.
        const int s = warp == 11, n_t = both || s == 0 ? n_t0 : n_t1;
        const uint32_t tmem_s = tmem + 256u * s, tmem_o = tmem_s + 128u;
        constexpr uint32_t idesc_s = make_idesc(TT_SIDE, TT_BN, false), idesc_o = make_idesc(TT_SIDE, D, true);
        const bool issuer = elect_one();
        const uint32_t q_full = q_full0 + 8 * s, s_full = s_full0 + 16 * s, p_full = p_full0 + 16 * s, p_free = p_free0 + 16 * s;
        const uint64_t qd = desc_k_major(sQ + s * TILE);
        // where this side's K and V tiles are in their rings, which of its tiles that is, and a bit a stage: the phase it waits for
        const uint32_t k_full = k_full0 + (both ? 0 : 8 * NK * s), v_full = v_full0 + (both ? 0 : 8 * NV * s);
        int ki = n_turns ? s : 0, vi = ki, kt = 0, vt = 0;
        uint32_t k_phase = 0, v_phase = 0;
        auto ahead = [&](int& i, int& t, int n) {
            i += stages_on(s, t);
            ++t;
            if (i >= n) i -= n;
        };
        auto k_seen = [&]() { k_phase ^= 1u << ki; };
        auto v_seen = [&]() { v_phase ^= 1u << vi; };
        int p_phase[2] = {0, 0}, q_phase = 0;
        TreeWalk w;
        if (n_t) w.at(a, st, both ? 0 : s);
        auto issue_s = [&](int half, bool last) {                     // K is there
            if (issuer) {
                const uint64_t kd = desc_k_major(sK0 + ki * TILE + half * SUB);
#pragma unroll
                for (int x = 0; x < PIECES; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma(tmem_s + (uint32_t)(half * TT_BN), qd + (PIECE >> 4) * x + 2u * k, kd + (PIECE >> 4) * x + 2u * k, idesc_s, x + k > 0 ? 1u : 0u);
                tc_commit(s_full + 8 * half);
                if (last) tc_commit(k_empty0 + 8 * ki);
            }
            __syncwarp();
        };
        bool ok = true;
        for (int done = 0; done < n_t && ok;) {                       // a part of an item
            const int nt = min(n_t - done, w.x.tiles - w.tile), row = (w.block() * (both ? 2 : 1) + (both ? s : 0)) * tile_rows;
            const int e0 = w.tile * TT_STAGE, e1 = min(w.x.entries, e0 + nt * TT_STAGE), n_kt = (e1 - e0 + TT_BN - 1) / TT_BN;
            if (row >= w.x.rows) {                                    // no queries on this side: give the tiles back
                for (int J = 0; J < nt && ok; ++J) {
                    ok = mbar_wait_all(k_full + 8 * ki, k_phase >> ki & 1, err, 73, &abort_flag);
                    if (ok && lane == 0) mbar_arrive(k_empty0 + 8 * ki);
                    if (ok) ok = mbar_wait_all(v_full + 8 * vi, v_phase >> vi & 1, err, 73, &abort_flag);
                    if (ok && lane == 0) mbar_arrive(v_empty0 + 8 * vi);
                    k_seen();
                    v_seen();
                    ahead(ki, kt, NK);
                    ahead(vi, vt, NV);
                }
            } else {
                // The last item's scores have all been read: its queries may go.
                if (lane == 0) mbar_expect_tx(q_full, (uint32_t)(PIECES * 128 * group * tile_rows));
                __syncwarp();
                if (lane < PIECES) tma_load_3d(sQ + s * TILE + lane * PIECE, &q_map, q_full, 64 * lane, w.kvh() * group, w.x.row0 + row);
                ok = wait_all_of(q_full, q_phase, k_full + 8 * ki, k_phase >> ki & 1, q_full, q_phase, err, 74, &abort_flag);
                q_phase ^= 1;
                k_seen();
                if (ok) { tc_fence_after(); issue_s(0, n_kt == 1); }
                if (ok && n_kt > 1) issue_s(1, true);                 // the same stage
                const int tail = e1 - e0 - (n_kt - 1) * TT_BN;        // entries of the last pass
                for (int J = 0; J < nt && ok; ++J) {
                    ahead(ki, kt, NK);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int j = 2 * J + half;
                        if (!ok || j >= n_kt) break;
                        const bool next = j + 2 < n_kt;
                        // this pass's weights, and once a tile V and the next tile's K: asked for together
                        const uint32_t p_bar = p_full + 8 * half;
                        if (half) ok = mbar_wait_all(p_bar, p_phase[1], err, 77, &abort_flag);
                        else {
                            ok = wait_all_of(p_bar, p_phase[0], v_full + 8 * vi, v_phase >> vi & 1, next ? k_full + 8 * ki : p_bar,
                                             next ? k_phase >> ki & 1 : p_phase[0], err, 76, &abort_flag);
                            v_seen();
                            if (next) k_seen();
                        }
                        if (!ok) break;
                        if (j == n_kt - 1 && tail < TT_BN) {
                            // rows of V behind the end may be anything: their weights are 0, and 0 times an infinity is no number
                            // (both sides may write the same zeros)
                            for (int i = lane; i < (TT_BN - tail) * 8 * PIECES; i += 32) {
                                const int key = tail + i / (8 * PIECES), c = i % (8 * PIECES);
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                                             ::"r"(sV0 + vi * TILE + half * SUB + (c >> 3) * PIECE + key * 128 + (c & 7) * 16), "r"(0) : "memory");
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the product reads them
                            __syncwarp();
                        }
                        p_phase[half] ^= 1;
                        tc_fence_after();
                        if (issuer) {
                            const uint64_t vd = desc_mn_major(sV0 + vi * TILE + half * SUB, PIECE);
#pragma unroll
                            for (int k = 0; k < TT_BN / 16; ++k)      // 16 entries: 16 rows of V, 8 cells of P
                                tc_mma_a_tmem(tmem_o, tmem_s + (uint32_t)(half * TT_BN + k * 8), vd + 128u * k, idesc_o, (j > 0 || k > 0) ? 1u : 0u);
                            tc_commit(p_free + 8 * half);
                            if (half == 1 || j == n_kt - 1) tc_commit(v_empty0 + 8 * vi);
                        }
                        __syncwarp();
                        // the scores of pass j + 2 over the scores and weights of this one: the tensor core takes them up after the
                        // product that reads them
                        if (next) issue_s(half, half == 1 || j + 2 == n_kt - 1);
                    }
                    ahead(vi, vt, NV);
                }
            }
            done += nt;
            w.next(a, done < n_t, nt);
        }
    } else if (warp < 8) {
        // ---- softmax and parts: thread = query
        const int s = warp >> 2, i = threadIdx.x & 127, n_t = both || s == 0 ? n_t0 : n_t1;
        const uint32_t tmem_sg = tmem + 256u * s + ((uint32_t)((warp & 3) * 32) << 16), tmem_o = tmem_sg + 128u;
        const uint32_t s_full = s_full0 + 16 * s, p_full = p_full0 + 16 * s, p_free = p_free0 + 16 * s;
        int s_phase = 0, o_phase = 0;                                 // bit `half`: of the next scores, of the next product
        TreeWalk w;
        if (n_t) w.at(a, st, both ? 0 : s);
        bool ok = true;
        for (int done = 0; done < n_t && ok;) {                       // a part of an item
            const int nt = min(n_t - done, w.x.tiles - w.tile), row_first = (w.block() * (both ? 2 : 1) + (both ? s : 0)) * tile_rows;
            const int e0 = w.tile * TT_STAGE, e1 = min(w.x.entries, e0 + nt * TT_STAGE), n_kt = row_first < w.x.rows ? (e1 - e0 + TT_BN - 1) / TT_BN : 0;
            const int row = row_first + i / group, t = w.x.row0 + row;
            const bool query = i < tile_rows * group && row < w.x.rows;
            const int plain = min(e1 - e0, max(0, w.x.start - e0)) / TT_BN;      // passes that everybody sees all of
            float m_ref = -INFINITY, l_run = 0.f;                     // reference maximum (log2 domain), row sum
            const bool idle = !__any_sync(0xffffffffu, query);        // a warp without queries only keeps the barriers going
            for (int j = 0; j < n_kt && ok; ++j) {
                const int half = j & 1, e = e0 + j * TT_BN, n = e1 - e;
                const uint32_t tmem_s = tmem_sg + (uint32_t)(half * TT_BN);
                ok = mbar_wait_all(s_full + 8 * half, s_phase >> half & 1, err, 78, &abort_flag);
                if (!ok) break;
                s_phase ^= 1 << half;
                tc_fence_after();
                if (idle) { mbar_arrive(p_full + 8 * half); o_phase ^= 1 << half; continue; }   // its lanes of P are scores: lanes have no say in one another
                const bool edge = j >= plain;
                uint64_t seen = ~0ull;
                if (edge) seen = query ? tree_seen(a, t, w.x.start, e, n) : 0ull;
                uint32_t pk[TT_BN / 2];
                auto exp_pass = [&](auto edge_c, float ms) -> float {
                    constexpr bool EDGE = decltype(edge_c)::value;
                    uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
                    const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2), nms2 = pack2(-ms, -ms);
                    uint32_t v[2][32];
                    tc_ld32_nowait(tmem_s, v[0]);
                    tc_ld32_nowait(tmem_s + 32u, v[1]);
                    tc_ld_wait();
                    // groups of 16 columns, consumers one group behind the exponentials (see attention_tcgen05.cu)
                    float p[2][16];
                    auto exps = [&](int c) {
#pragma unroll
                        for (int x = 0; x < 16; x += 2) {
                            const int col = c * 16 + x;
                            float s0 = __uint_as_float(v[col >> 5][col & 31]), s1 = __uint_as_float(v[col >> 5][(col & 31) + 1]);
                            if (EDGE) {
                                if (!(seen >> col & 1)) s0 = -INFINITY;
                                if (!(seen >> (col + 1) & 1)) s1 = -INFINITY;
                            }
                            float t0, t1;
                            unpack2(fma2(pack2(s0, s1), scale2, nms2), t0, t1);
                            p[c & 1][x] = ex2_in_order(t0);
                            p[c & 1][x + 1] = ex2_in_order(t1);
                        }
                    };
                    auto consume = [&](int c) {
#pragma unroll
                        for (int x = 0; x < 16; x += 2) {
                            rs2[(x >> 1) & 3] = add2_in_order(rs2[(x >> 1) & 3], pack2(p[c & 1][x], p[c & 1][x + 1]));
                            pk[c * 8 + (x >> 1)] = bf16x2_in_order(p[c & 1][x], p[c & 1][x + 1]);
                        }
                    };
                    exps(0);
                    exps(1);
                    consume(0);
                    exps(2);
                    consume(1);
                    exps(3);
                    consume(2);
                    consume(3);
                    float x, y;
                    unpack2(add2(add2(rs2[0], rs2[1]), add2(rs2[2], rs2[3])), x, y);
                    return x + y;
                };
                auto pass = [&](float ms) -> float { return edge ? exp_pass(std::true_type{}, ms) : exp_pass(std::false_type{}, ms); };
                bool redo = j == 0, mine = redo;                      // mine: this query's reference moves; the warp's others keep theirs
                float row_sum = 0.f;
                if (!redo) {
                    row_sum = pass(m_ref == -INFINITY ? 0.f : m_ref);
                    mine = query && (!(row_sum <= 256.f) || m_ref == -INFINITY);   // inf and NaN, too
                    redo = __any_sync(0xffffffffu, mine);
                }
                if (redo) {
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // on raw scores: the scale is positive
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t v[32];
                        tc_ld32(tmem_s + 32u * c, v);
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (seen >> (32 * c + x) & 1) mx4[x & 3] = fmaxf(mx4[x & 3], __uint_as_float(v[x]));
                    }
                    const float m_new = mine ? fmaxf(m_ref, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2) : m_ref;
                    if (j > 0) {
                        // O must be complete through pass j - 1 (the product of pass j waits for this pass's P)
                        ok = mbar_wait_all(p_free + 8 * (half ^ 1), (o_phase >> (half ^ 1) & 1) ^ 1, err, 79, &abort_flag);
                        if (!ok) break;
                        tc_fence_after();
                        const float alpha = ex2(m_ref - (m_new == -INFINITY ? 0.f : m_new));
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tc_ld32(tmem_o + (uint32_t)(c * 32), o);
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                            tc_st32(tmem_o + (uint32_t)(c * 32), o);
                        }
                        tc_st_wait();
                        l_run *= alpha;
                    }
                    m_ref = m_new;
                    row_sum = pass(m_ref == -INFINITY ? 0.f : m_ref);
                }
                l_run += row_sum;
                tc_st32(tmem_s, pk);
                tc_st_wait();
                tc_fence_before();
                mbar_arrive(p_full + 8 * half);                       // this query's scores have been read, its weights written
                o_phase ^= 1 << half;
            }
            if (ok && n_kt > 0 && !idle) {
                const int half = (n_kt - 1) & 1;
                ok = mbar_wait_all(p_free + 8 * half, (o_phase >> half & 1) ^ 1, err, 79, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                const size_t place = (size_t)w.first_query(a) + (size_t)worker_of(s) * a.item_queries + (both ? s * tile_rows * group : 0) + i;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tc_ld32(tmem_o + (uint32_t)(c * 32), o);          // every lane takes part in the load
                    if (query)
#pragma unroll
                        for (int x = 0; x < 32; x += 8) tt_store8(a.part_o + place * D + c * 32 + x, o, x);
                }
                if (query) {
                    *reinterpret_cast<float2*>(a.part_ml + place * 2) = make_float2(m_ref, l_run);
                    if (w.tile == 0) a.parts[(size_t)t * a.nh + w.kvh() * group + i % group] = make_int2((int)place, w.parts(st.per));
                }
                tc_fence_before();                                    // before the next item's first product
            }
            done += nt;
            w.next(a, done < n_t, nt);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {                                                 // give copies in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 11) {
        tc_fence_after();
        tmem_free(tmem, 512u);
    }
}

// bfloat16, head sizes 64 and 128, up to 128 heads a kv head, pages of 8 tokens or a larger power of two, rows of q on 16-byte
// boundaries, and addresses that fit the maps' coordinates.
static bool tree_tc_ok(const TreeArgs& a, int dtype) {
    return dtype == RG_DTYPE_BF16 && (a.d == 64 || a.d == 128) && a.nh / a.nkv <= TT_SIDE && a.page_shift >= 3 && a.q_stride % 8 == 0 &&
           (((uintptr_t)a.q | (uintptr_t)a.kv) & 15) == 0 && ((uintptr_t)a.part_o & 31) == 0 && a.scale_log2 > 0.f && a.max_blocks > 0 &&
           (long long)a.pages * 2 * a.nkv * a.page_size < 0x7fffffffll;
}

// blocks: one to an SM; a.item_queries: tile_rows x heads of a kv head, twice that with `both`.
static int launch_tree_tc(const TreeArgs& a, int tile_rows, int both, int blocks, cudaStream_t s) {
    const int group = a.nh / a.nkv;
    if (tile_rows < 1 || tile_rows * group > TT_SIDE || a.item_queries != tile_rows * group * (both ? 2 : 1) || a.workers != blocks * (both ? 1 : 2))
        return RG_ERR_UNSUPPORTED;
    RgEncodeTiledFn fn = rg_encode_fn();
    if (!fn) return RG_ERR_UNSUPPORTED;
    CUtensorMap qm, km;
    cuuint64_t dims[3] = {(cuuint64_t)a.d, (cuuint64_t)a.nh, (cuuint64_t)a.T}, strides[2] = {(cuuint64_t)a.d * 2, (cuuint64_t)a.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tile_rows}, estr[3] = {1, 1, 1};
    CUresult r = fn(&qm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return 20000 + (int)r;
    int e = rg_make_map(&km, a.kv, (unsigned long long)a.pages * 2 * a.nkv * a.page_size, a.d, a.d, a.page_size < TT_STAGE ? a.page_size : TT_STAGE);
    if (e) return e;
#define RG_TT(P) { RG_ALLOW_SMEM(tree_tc_kernel<P>, tt_smem(P)) \
    return rg_launch(tree_tc_kernel<P>, dim3((unsigned)blocks), dim3(TT_THREADS), (size_t)tt_smem(P), s, 1, qm, km, a, tile_rows, both); }
    if (a.d == 64) RG_TT(1)
    RG_TT(2)
#undef RG_TT
}
