// Attention of single tokens over prefixes that rows share, on the 5th-generation tensor cores (bfloat16, head sizes 64
// and 128): the parts of prefixes that attention_parts.cuh describes, for many queries a kv head.
//
// A block takes one part of a prefix and up to 256 queries (rows x heads of a kv head) as two sides of 128, each with
// its own softmax threads, accumulator and issuing warp; K and V tiles of 128 entries (TMA through the prefix's table, one
// box a page and 64 columns, 128-byte swizzle) are fetched once for both.  With up to 128 queries the sides take a part
// each of their own instead, so that two chains of scores, exponentials and products are under way on the SM either way.
// Per side and 64 entries j:
//   S(j) = Q K^T         tcgen05.mma, M 128 x N 64 x K head size, into one of two buffers of 64 TMEM columns
//   softmax              128 threads, one query each; the reference maximum is raised only when the 64 weights sum to more than 2^8
//   O += P(j) V          tcgen05.mma, M 128 x N head size x K 64: P as bfloat16 in TMEM over the scores it was made from
// S(j + 2) is issued behind O += P(j) V, which reads the buffer that it goes to, so S(j + 1) is there when the threads are done
// with j: the exponentials never wait for a product of their own side.  (With one buffer of 128 columns and N 128, the faster
// shape by 260 to 392 cycles for 64 entries, a side's scores, exponentials and products are one chain: 65,536 entries for
// 512 queries a kv head 189 us, 171 with two.)
// What bounds it: 65,536 entries for 128 rows of 32 heads on 8 of 128 take 155 us with the rows' 256 own entries beside them, 1,010
// TFLOP/s while the tiles run (59 % of what a dense product reaches): N 64 scores cost the tensor core 49 cycles where 33 would
// do, and the hand-over between products and exponentials the rest.
// There is no mask but the end of a part: rows of V behind it get zeros in shared memory, scores behind it -infinity.
//
// Rounding: P to bfloat16 (up to 2^-8 of each weight; the sum of weights is of the unrounded ones), all sums in 32-bit.
#pragma once
#include "attention_parts.cuh"
#include "packed_f32.cuh"
#include "tcgen05.cuh"
#include <type_traits>

#define PT_SIDE 128                // queries of a side
#define PT_BN 64                   // entries of a softmax pass
#define PT_STAGE 128               // entries of a K or V stage
#define PT_THREADS 384             // warps 0-3, 4-7: softmax of side 0, 1; 8, 10: TMA of K (and Q), of V; 9, 11: MMA issue of side 0, 1
#define PT_BARRIERS 384            // bytes
__host__ __device__ constexpr int pt_k_stages(int pieces) { return pieces == 1 ? 5 : 3; }
__host__ __device__ constexpr int pt_v_stages(int pieces) { return pieces == 1 ? 4 : 2; }
__host__ __device__ constexpr int pt_smem(int pieces) {
    return (2 + pt_k_stages(pieces) + pt_v_stages(pieces)) * PT_SIDE * 128 * pieces + PT_BARRIERS + 1024;
}

__device__ __forceinline__ void store8(float* p, const uint32_t (&v)[32], int i) {      // 32 bytes: a whole sector of the row
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]),
                 "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7]) : "memory");
}

// q_map: 64 columns x heads x rows, a box of 64 x group x tile_rows (tile_rows = 128 / group rows fill a side); kv_map: the
// cache as rows of the head size, a box of min(page, 128) rows x 64 columns.  two_parts: the sides take a part each.
template <int PIECES>
__global__ void __launch_bounds__(PT_THREADS, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const PartArgs a, int tile_rows,
                 int two_parts, int* err) {
    extern __shared__ unsigned char smem_raw[];
    constexpr int D = 64 * PIECES, NK = pt_k_stages(PIECES), NV = pt_v_stages(PIECES);
    constexpr uint32_t PIECE = PT_STAGE * 128, TILE = PIECE * PIECES, SUB = PT_BN * 128;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t sQ = base, sK0 = sQ + 2 * TILE, sV0 = sK0 + NK * TILE, bars = sV0 + NV * TILE;
    // A stage is full on the barrier of the side whose tile it holds (side 0's, where the tile is both sides').  A wait goes by the parity of
    // a phase, so that who waits has to have seen all phases before: of barriers that both sides' tiles came through in turn, a side would
    // see every second one, and take its tile for loaded while the other side's before it was still on its way.
    const uint32_t q_full = bars, k_full0 = bars + 8, k_empty0 = k_full0 + 16 * NK, v_full0 = k_empty0 + 8 * NK, v_empty0 = v_full0 + 16 * NV,
                   s_full0 = v_empty0 + 8 * NV, p_full0 = s_full0 + 32, p_free0 = p_full0 + 32;    // per side and half stage
    static_assert(8 + 24 * (NK + NV) + 32 + 64 <= PT_BARRIERS, "the barriers' place");
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.nh / a.nkv;
    // block = (prefix, kv head, 256 queries or 128, part or pair of parts), parts innermost
    const int sides = two_parts ? 1 : 2, grid_parts = two_parts ? (a.prefix_parts + 1) / 2 : a.prefix_parts;
    const int part = blockIdx.x % grid_parts, rest = blockIdx.x / grid_parts, blk = rest % a.prefix_tiles, gk = rest / a.prefix_tiles;
    const int g_id = gk / a.nkv, kvh = gk % a.nkv;
    pdl_wait();                                                      // tables, lengths and queries may come from the kernel before
    pdl_trigger();
    const int row0 = a.groups[g_id * 3], entries = prefix_entries(a, g_id);
    const int rows = group_rows(a, g_id);
    const int tile0 = blk * sides;                                    // of tile_rows rows each
    // what side s looks at: its part's entries [e0, e1), in passes of 64 and stages of 128
    auto first_of = [&](int s) -> int { return (two_parts ? 2 * part + s : part) * a.prefix_per; };
    auto end_of = [&](int s) -> int { return min(entries, first_of(s) + a.prefix_per); };
    auto passes_of = [&](int s) -> int {
        const int left = rows - (two_parts ? tile0 : tile0 + s) * tile_rows;
        return left <= 0 ? 0 : max(0, end_of(s) - first_of(s) + PT_BN - 1) / PT_BN;
    };
    const int n_kt0 = passes_of(0), n_kt1 = passes_of(1), n_st0 = (n_kt0 + 1) / 2, n_st1 = (n_kt1 + 1) / 2;
    if (n_kt0 == 0) return;                                           // nothing for side 0: nothing at all
    // A stage of the stream belongs to both sides, or in turn to either while side 1 has some
    const int n_stages = two_parts ? n_st0 + n_st1 : n_st0;

    if (threadIdx.x == 0) {
        const uint32_t users = two_parts || n_kt1 == 0 ? 1 : 2;
        abort_flag = 0;
        mbar_init(q_full, 1);
        for (int s = 0; s < 2 * NK; ++s) mbar_init(k_full0 + 8 * s, 1);
        for (int s = 0; s < 2 * NV; ++s) mbar_init(v_full0 + 8 * s, 1);
        for (int s = 0; s < NK; ++s) mbar_init(k_empty0 + 8 * s, users);
        for (int s = 0; s < NV; ++s) mbar_init(v_empty0 + 8 * s, users);
        for (int b = 0; b < 4; ++b) { mbar_init(s_full0 + 8 * b, 1); mbar_init(p_full0 + 8 * b, PT_SIDE); mbar_init(p_free0 + 8 * b, 1); }
        fence_barrier_init();
    }
    if (warp == 9) tmem_alloc(&tmem_base_slot, 512u);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // side s: scores and weights in columns [256 s, 256 s + 128), O in [256 s + 128, 256 s + 128 + D)
    const uint32_t tmem = tmem_base_slot;

    if (warp == 8 || warp == 10) {
        // ---- producers of K and of V.  A stage is 128 / box_rows boxes for each 64 columns; lane l has box l % boxes of piece l / boxes.
        const int box_rows = min(a.page_size, PT_STAGE), boxes = PT_STAGE / box_rows, box = lane % boxes, piece = lane / boxes;
        const bool mine = piece < PIECES;
        const int* table = a.prefix_table + (size_t)g_id * a.prefix_blocks;
        auto tile_of = [&](int b, int& s, int& J) {                   // the side (or 0) and tile of stage b
            if (!two_parts) { s = 0; J = b; }
            else if (b < 2 * n_st1) { s = b & 1; J = b >> 1; }
            else { s = 0; J = b - n_st1; }
        };
        auto page_of = [&](int b) -> int {                            // behind the part: any page
            int s, J;
            tile_of(b, s, J);
            const int e = first_of(s) + J * PT_STAGE + box * box_rows;
            return b < n_stages ? table[(e < end_of(s) ? e : first_of(s)) >> a.page_shift] : 0;
        };
        const int kv = warp == 10 ? 1 : 0, n = kv ? NV : NK;
        if (kv == 0 && lane == 0) mbar_expect_tx(q_full, (uint32_t)((n_kt1 && !two_parts ? 2 : 1) * PIECES * 128 * group * tile_rows));
        __syncwarp();
        if (kv == 0 && lane < 2 * PIECES) {
            const int s = lane / PIECES, x = lane % PIECES;
            if (s == 0 || (n_kt1 && !two_parts))
                tma_load_3d(sQ + s * TILE + x * PIECE, &q_map, q_full, 64 * x, kvh * group, row0 + (tile0 + s) * tile_rows);
        }
        int page_next = page_of(0);
        bool ok = true;
        for (int b = 0; b < n_stages && ok; ++b) {
            int s, J;
            tile_of(b, s, J);
            const int page = page_next, e = first_of(s) + J * PT_STAGE + box * box_rows, in_page = e & (a.page_size - 1);
            page_next = page_of(b + 1);
            const int st = b % n, u = b / n;
            const uint32_t full = (kv ? v_full0 : k_full0) + 8 * (st + n * s), empty = (kv ? v_empty0 : k_empty0) + 8 * st;
            if (u > 0) ok = mbar_wait_all(empty, (u & 1) ^ 1, err, 51 + kv, &abort_flag);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(full, TILE);
            __syncwarp();
            if (mine)
                tma_load_2d((kv ? sV0 : sK0) + st * TILE + piece * PIECE + box * box_rows * 128, &kv_map, full, 64 * piece,
                            ((page * 2 + kv) * a.nkv + kvh) * a.page_size + in_page);
        }
    } else if (warp == 9 || warp == 11) {
        // ---- MMA issue of one side.  The whole warp walks the loop and waits; one elected lane issues.  The loop is lean: its
        // instructions share a scheduler with two warps of exponentials, and what it does between two products is time that
        // the tensor core may stand still.
        const int s = warp == 11, n_kt = s ? n_kt1 : n_kt0, n_st = (n_kt + 1) >> 1;
        const uint32_t tmem_s = tmem + 256u * s, tmem_o = tmem_s + 128u;
        constexpr uint32_t idesc_s = make_idesc(PT_SIDE, PT_BN, false), idesc_o = make_idesc(PT_SIDE, D, true);
        const bool issuer = elect_one();
        const uint64_t qd = desc_k_major(sQ + (two_parts ? 0 : s) * TILE);
        // where this side's K and V tiles are in their rings, `step` stages of the stream from one to the next
        const uint32_t k_full = k_full0 + (two_parts ? 8 * NK * s : 0), v_full = v_full0 + (two_parts ? 8 * NV * s : 0);
        int ki = two_parts ? s : 0, vi = ki;
        uint32_t k_phase = 0, v_phase = 0;                            // a bit a stage: the phase that this side waits for
        auto step = [&](int J) -> int { return two_parts && (s || J < n_st1) ? 2 : 1; };   // from tile J to tile J + 1
        auto ahead = [&](int& i, uint32_t& phase, int by, int n) {    // from a stage that has been waited for
            phase ^= 1u << i;
            i += by;
            if (i >= n) i -= n;
        };
        auto issue_s = [&](int half, bool last) {                     // the next pass's scores: K is there
            if (issuer) {
                const uint64_t kd = desc_k_major(sK0 + ki * TILE + half * SUB);
#pragma unroll
                for (int x = 0; x < PIECES; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc_mma(tmem_s + (uint32_t)(half * PT_BN), qd + (PIECE >> 4) * x + 2u * k, kd + (PIECE >> 4) * x + 2u * k, idesc_s, x + k > 0 ? 1u : 0u);
                tc_commit(s_full0 + 16 * s + 8 * half);
                if (last) tc_commit(k_empty0 + 8 * ki);
            }
            __syncwarp();
        };
        bool ok = n_kt > 0;
        if (ok) ok = mbar_wait_all(q_full, 0, err, 53, &abort_flag);
        if (ok) ok = mbar_wait_all(k_full + 8 * ki, 0, err, 54, &abort_flag);
        if (ok) { tc_fence_after(); issue_s(0, n_kt == 1); }
        if (ok && n_kt > 1) issue_s(1, true);                         // the same stage
        const int tail = end_of(s) - first_of(s) - (n_kt - 1) * PT_BN;    // entries of the last pass
        for (int J = 0; J < n_st && ok; ++J) {
            ok = mbar_wait_all(v_full + 8 * vi, v_phase >> vi & 1, err, 55, &abort_flag);
            if (J + 1 < n_st) ahead(ki, k_phase, step(J), NK);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int j = 2 * J + half;
                if (!ok || j >= n_kt) break;
                if (j == n_kt - 1 && tail < PT_BN) {
                    // rows of V behind the part may be anything: their weights are 0, and 0 times an infinity is no number (both
                    // sides may write the same zeros)
                    for (int i = lane; i < (PT_BN - tail) * 8 * PIECES; i += 32) {
                        const int key = tail + i / (8 * PIECES), c = i % (8 * PIECES);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                                     ::"r"(sV0 + vi * TILE + half * SUB + (c >> 3) * PIECE + key * 128 + (c & 7) * 16), "r"(0) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the product reads them
                    __syncwarp();
                }
                const bool next = j + 2 < n_kt;
                if (half == 0 && next) ok = mbar_wait_all(k_full + 8 * ki, k_phase >> ki & 1, err, 54, &abort_flag);
                if (ok) ok = mbar_wait_all(p_full0 + 16 * s + 8 * half, J & 1, err, 56, &abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (issuer) {
                    const uint64_t vd = desc_mn_major(sV0 + vi * TILE + half * SUB, PIECE);
#pragma unroll
                    for (int k = 0; k < PT_BN / 16; ++k)              // 16 entries: 16 rows of V, 8 cells of P
                        tc_mma_a_tmem(tmem_o, tmem_s + (uint32_t)(half * PT_BN + k * 8), vd + 128u * k, idesc_o, (j > 0 || k > 0) ? 1u : 0u);
                    tc_commit(p_free0 + 16 * s + 8 * half);
                    if (half == 1 || j == n_kt - 1) tc_commit(v_empty0 + 8 * vi);
                }
                __syncwarp();
                // the scores of pass j + 2 over the scores and weights of this one: the tensor core takes them up after the product
                // that reads them
                if (next) issue_s(half, half == 1 || j + 2 == n_kt - 1);
            }
            ahead(vi, v_phase, step(J), NV);
        }
    } else if (warp < 8 && (warp < 4 || n_kt1 > 0)) {
        // ---- softmax and output: thread = query
        const int s = warp >> 2, i = threadIdx.x & 127, n_kt = s ? n_kt1 : n_kt0;
        const int row = (two_parts ? tile0 : tile0 + s) * tile_rows + i / group;
        const bool query = i < tile_rows * group && row < rows;
        const int e0 = first_of(s), e1 = end_of(s);
        const uint32_t tmem_sg = tmem + 256u * s + ((uint32_t)((warp & 3) * 32) << 16), tmem_o = tmem_sg + 128u;
        const uint32_t p_full = p_full0 + 16 * s, p_free = p_free0 + 16 * s;
        float m_ref = -INFINITY, l_run = 0.f;                         // reference maximum (log2 domain), row sum
        const bool idle = !__any_sync(0xffffffffu, query);            // a warp without queries only keeps the barriers going
        bool ok = true;
        for (int j = 0; j < n_kt && ok; ++j) {
            const int J = j >> 1, half = j & 1, n = e1 - e0 - j * PT_BN;
            const uint32_t tmem_s = tmem_sg + (uint32_t)(half * PT_BN);
            ok = mbar_wait_all(s_full0 + 16 * s + 8 * half, J & 1, err, 57, &abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (idle) { mbar_arrive(p_full + 8 * half); continue; }   // its lanes of P are scores: lanes have no say in one another
            uint32_t pk[PT_BN / 2];
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
                            if (col >= n) s0 = -INFINITY;
                            if (col + 1 >= n) s1 = -INFINITY;
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
            auto pass = [&](float ms) -> float { return n < PT_BN ? exp_pass(std::true_type{}, ms) : exp_pass(std::false_type{}, ms); };
            bool redo = j == 0;
            float row_sum = 0.f;
            if (!redo) {
                row_sum = pass(m_ref == -INFINITY ? 0.f : m_ref);
                redo = __any_sync(0xffffffffu, query && (!(row_sum <= 256.f) || m_ref == -INFINITY));   // inf and NaN, too
            }
            if (redo) {
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};   // on raw scores: the scale is positive
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[32];
                    tc_ld32(tmem_s + 32u * c, v);
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (32 * c + x < n) mx4[x & 3] = fmaxf(mx4[x & 3], __uint_as_float(v[x]));
                }
                const float m_new = fmaxf(m_ref, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2);
                if (j > 0) {
                    // O must be complete through pass j - 1 (the product of pass j waits for this pass's P)
                    ok = mbar_wait_all(p_free + 8 * ((j - 1) & 1), ((j - 1) >> 1) & 1, err, 58, &abort_flag);
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
            mbar_arrive(p_full + 8 * half);                           // this query's scores have been read, its weights written
        }
        if (ok) ok = mbar_wait_all(p_free + 8 * ((n_kt - 1) & 1), ((n_kt - 1) >> 1) & 1, err, 59, &abort_flag);
        if (ok) {
            tc_fence_after();
            const int slots = a.prefix_parts + a.own_parts, slot = two_parts ? 2 * part + s : part;
            const size_t place = ((size_t)(row0 + row) * a.nh + kvh * group + i % group) * slots + slot;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tc_ld32(tmem_o + (uint32_t)(c * 32), o);              // every lane takes part in the load
                if (query)
#pragma unroll
                    for (int x = 0; x < 32; x += 8) store8(a.part_o + place * D + c * 32 + x, o, x);
            }
            if (query) *reinterpret_cast<float2*>(a.part_ml + place * 2) = make_float2(m_ref, l_run);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {                                                 // give copies in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 9) {
        tc_fence_after();
        tmem_free(tmem, 512u);
    }
}

// bfloat16, head sizes 64 and 128, up to 128 heads a kv head, pages of 8 tokens or a larger power of two, rows of q on 16-byte
// boundaries, and addresses that fit the maps' coordinates.
static bool prefix_tc_ok(const PartArgs& a, int dtype, int num_pages) {
    return dtype == RG_DTYPE_BF16 && (a.d == 64 || a.d == 128) && a.nh / a.nkv <= PT_SIDE && a.page_shift >= 3 && a.q_stride % 8 == 0 &&
           (((uintptr_t)a.q | (uintptr_t)a.kv) & 15) == 0 && ((uintptr_t)a.part_o & 31) == 0 && a.scale_log2 > 0.f &&
           a.prefix_per % PT_STAGE == 0 && (long long)num_pages * 2 * a.nkv * a.page_size < 0x7fffffffll;
}

// The prefixes' parts; a.prefix_tiles: the blocks of 256 queries of a group, or of 128 with two_parts.
static int launch_prefix_tc(const PartArgs& a, int num_pages, int two_parts, int* err, cudaStream_t s) {
    const int group = a.nh / a.nkv, tile_rows = PT_SIDE / group;
    const long long blocks = (long long)a.n_groups * a.nkv * a.prefix_tiles * (two_parts ? (a.prefix_parts + 1) / 2 : a.prefix_parts);
    if (blocks > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
    if (blocks == 0) return 0;
    RgEncodeTiledFn fn = rg_encode_fn();
    if (!fn) return RG_ERR_UNSUPPORTED;
    CUtensorMap qm, km;
    cuuint64_t dims[3] = {(cuuint64_t)a.d, (cuuint64_t)a.nh, (cuuint64_t)a.T}, strides[2] = {(cuuint64_t)a.d * 2, (cuuint64_t)a.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tile_rows}, estr[3] = {1, 1, 1};
    CUresult r = fn(&qm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return 20000 + (int)r;
    int e = rg_make_map(&km, a.kv, (unsigned long long)num_pages * 2 * a.nkv * a.page_size, a.d, a.d, a.page_size < PT_STAGE ? a.page_size : PT_STAGE);
    if (e) return e;
#define RG_PT(P) { RG_ALLOW_SMEM(prefix_tc_kernel<P>, pt_smem(P)) \
    return rg_launch(prefix_tc_kernel<P>, dim3((unsigned)blocks), dim3(PT_THREADS), (size_t)pt_smem(P), s, 1, qm, km, a, tile_rows, two_parts, err); }
    if (a.d == 64) RG_PT(1)
    RG_PT(2)
#undef RG_PT
}
