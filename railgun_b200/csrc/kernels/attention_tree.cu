// Attention of trees of drafted tokens over the paged cache and over one another.  attention_tree.cuh says what is computed and
// how it is cut.
#include "attention_tree.cuh"
#include "attention_tree_rows.cuh"
#include "attention_tree_tcgen05.cuh"
#include "mma.cuh"

#define TG_THREADS 128
#define TG_Q 16                // queries of an item
#define TG_K 64                // entries of a tile
#define TG_LD (TG_K + 4)
// Places in front of an item's tiles.  In 32-bit, 16 heads on 4, with 0, 1 and 2 of them: 16 requests of 16 nodes behind up to 700 entries
// (128) 88.5, 83.4 and 89.7 us, 4 of 64 on 2,000 (64) 156.5, 154.5 and 160.5, 64 of 4 behind up to 300 (128) 68.4, 68.8 and 73.7.
#define TG_BEGIN 1

template <typename A> struct Quad;                                  // four numbers of a row at once
template <> struct Quad<float> {
    __device__ static float4 load(const float* p) { return *reinterpret_cast<const float4*>(p); }
};
template <> struct Quad<bf16> {
    __device__ static float4 load(const bf16* p) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
                           __uint_as_float(v.y & 0xffff0000u));
    }
};

__host__ __device__ constexpr int tg_row(int d) { return ((d + 3) & ~3) + 4; }   // floats a row in shared memory
__host__ __device__ inline int tg_stages(int d) { return d <= 128 ? 2 : 1; }   // tiles of K and V in shared memory: the next one is on its way
// Floats of a stage: a tile's K and V, and no fewer than the sums that go through it where an item ends and groups of threads share the
// columns (d up to 64), since the next stage then holds the next item's first tile already.  Heads of 1 to 8 have tiles of fewer.
#define TG_SUMS (TG_Q * TG_THREADS)
__host__ __device__ constexpr int tg_stage(int d) {
    const int tile = 2 * TG_K * tg_row(d);
    return d <= 64 && tile < TG_SUMS ? TG_SUMS : tile;
}
static_assert(tg_stage(1) >= TG_SUMS && tg_stage(8) >= TG_SUMS && tg_stage(9) >= TG_SUMS && tg_stage(64) >= TG_SUMS, "the groups' sums fit a stage");
static_assert(2 * tg_stage(1) >= TG_SUMS + TG_Q && 2 * tg_stage(32) >= TG_SUMS + TG_Q * 32 && 2 * tg_stage(64) >= TG_SUMS + TG_Q * 64,
              "and behind a cluster's results both stages");

// ---------------------------------------------------------------------------------------------------
// Any head size up to 256, any page size, 32-bit or bfloat16 storage, all arithmetic in 32-bit.
// Per tile of 64 entries: 2 queries x 4 entries of scores a thread, then a column of the output for all 16 queries a thread;
// DP = 32 or 64: as many threads share the columns, and TG_THREADS / DP groups of them share the tile's entries.
// WHOLE: an item to a cluster, whose blocks share its tiles, join through each other's shared memory and leave the output.
// What bounds it is shared memory: 96 bytes a thread for 32 products of scores, 272, most of them the same for a warp, for 64 of the output: in
// 32-bit, 16 heads on 4 of 128, one request of 16 nodes on 1,000 entries takes 26 us, 8 on 4,000 390, 10.7 TFLOP/s.  Smallest calls are the launch and
// three trips to memory, for the request, the table and the entries: two requests of 7 nodes on 61 entries, 3 heads on 1 of 32, 9.3 us in one launch, 12 in two.
// ---------------------------------------------------------------------------------------------------
template <typename A, int DP, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(TG_THREADS) tree_general_kernel(const TreeArgs a, A* __restrict__ out, int out_ld, int q_blocks) {
    extern __shared__ __align__(16) float smem[];
    constexpr int GROUPS = TG_THREADS / DP, COLS = DP == 128 ? 2 : 1;
    __shared__ TreeStart st;
    __shared__ long long row_at[2][TG_K];                           // where the rows of a tile are in the cache, -1 behind its end
    pdl_wait();
    pdl_trigger();
    TreeWalk w, ahead;                                              // this tile, and the one whose rows are looked up
    int n_tiles, C = 1, rank = 0;
    if constexpr (WHOLE) {
        C = cg::this_cluster().num_blocks();
        rank = cg::this_cluster().block_rank();
        if (!tree_item(a, blockIdx.x / C, q_blocks, w)) return;      // all blocks of the cluster
        const int per = (w.x.tiles + C - 1) / C;
        w.tile = min(w.x.tiles, rank * per);
        n_tiles = min(w.x.tiles, w.tile + per) - w.tile;
    } else {
        tree_plan<TG_THREADS>(a, blockIdx.x, 1, 0, st);
        n_tiles = st.tiles(0);
        if (n_tiles == 0) return;
        w.at(a, st, 0);
    }
    const int d = a.d, ld = tg_row(d), group = a.nh / a.nkv, tid = threadIdx.x, stages = tg_stages(d);
    float* qs = smem;                                               // [16][ld]
    const int stage = tg_stage(d);
    float* kv0 = qs + TG_Q * ld;                                    // [stages][K [64][ld], V [64][ld]], `stage` floats each
    float* ps = kv0 + stages * stage;                               // [16][TG_LD]
    float* al = ps + TG_Q * TG_LD;                                  // [16]
    const size_t to_values = (size_t)a.nkv * a.page_size * d;
    ahead = w;
    int looked = 0;
    auto look_up = [&](int slot) {                                  // of the next tile that has not been; the whole block
        if (tid < TG_K) {
            const int e = ahead.tile * TG_K + tid;
            row_at[slot][tid] = looked < n_tiles && e < ahead.x.entries ? entry_at(a, ahead.r, ahead.kvh(), e) : -1;
        }
        if (looked < n_tiles) ahead.next(a, ++looked < n_tiles);
    };
    // a thread's pieces of a tile: every 128th
    const int pieces = VEC ? d / 4 : d, row_first = tid / pieces, piece_first = tid - row_first * pieces, row_step = TG_THREADS / pieces,
              piece_step = TG_THREADS - row_step * pieces;
    auto request = [&](int slot, float* ks) {                       // rows behind the end are zeros
        constexpr int W = VEC ? 4 : 1;
        float* vs = ks + TG_K * ld;
        for (int row = row_first, p = piece_first; row < TG_K; p += piece_step, row += row_step) {
            if (p >= pieces) { p -= pieces; if (++row >= TG_K) break; }
            const int c = p * W;
            const long long at = row_at[slot][row];
            const A* src = (const A*)a.kv + (at < 0 ? 0 : at + c);
            if constexpr (VEC && sizeof(A) == 4) {
                rgmma::cp_async16(ks + row * ld + c, src, at >= 0);
                rgmma::cp_async16(vs + row * ld + c, src + (at < 0 ? 0 : to_values), at >= 0);
            } else {
                float4 k4 = {0.f, 0.f, 0.f, 0.f}, v4 = k4;
                if (at >= 0) {
                    if constexpr (VEC) { k4 = Quad<A>::load(src); v4 = Quad<A>::load(src + to_values); }
                    else { k4.x = to_f32(src[0]); v4.x = to_f32(src[to_values]); }
                }
                if constexpr (VEC) {
                    *reinterpret_cast<float4*>(ks + row * ld + c) = k4;
                    *reinterpret_cast<float4*>(vs + row * ld + c) = v4;
                } else { ks[row * ld + c] = k4.x; vs[row * ld + c] = v4.x; }
            }
        }
        if (!VEC)                                                   // the scores read four columns at a time
            for (int i = tid; i < TG_K * (ld - d); i += TG_THREADS) ks[i / (ld - d) * ld + d + i % (ld - d)] = 0.f;
        rgmma::cp_async_commit();
    };
    const int qa = tid >> 4, ka = tid & 15;                         // scores: queries 2 qa, 2 qa + 1; entries ka + 16 j
    const int col = tid % DP, part = tid / DP;                      // output: column(s) col (+ 128), entries part + GROUPS j
    float m[2], l[2];
    float acc[COLS][TG_Q];
    int q0 = 0, nq = 0, parts = 0;                                  // parts of the item, 0: it began before this stretch
    auto begin = [&]() {                                            // an item
        q0 = w.block() * TG_Q;
        nq = min(TG_Q, w.x.rows * group - q0);
        if constexpr (!WHOLE) parts = w.tile == 0 ? w.parts(st.per) : 0;
        for (int j = tid; j < TG_Q * ld; j += TG_THREADS) {         // nobody reads the last item's any more
            const int row = j / ld, c = j - row * ld, qi = q0 + row;
            float v = 0.f;
            if (row < nq && c < d)
                v = to_f32(((const A*)a.q)[(size_t)(w.x.row0 + qi / group) * a.q_stride + (w.kvh() * group + qi % group) * d + c]) * a.scale_log2;
            qs[j] = v;
        }
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int j = 0; j < TG_Q; ++j) acc[c][j] = 0.f;
    };
    look_up(0);
    look_up(1);
    __syncthreads();
    if (stages == 2 && n_tiles > 0) request(0, kv0);
    if (WHOLE) begin();
    for (int step = 0; step < n_tiles; ++step) {
        if (!WHOLE && (step == 0 || w.tile == 0)) begin();
        const int slot = step & 1, e0 = w.tile * TG_K, n = min(TG_K, w.x.entries - e0);
        float* ks = kv0 + (stages == 2 ? slot * stage : 0);
        const float* vs = ks + TG_K * ld;
        if (stages == 1) {
            __syncthreads();                                        // the last tile's values are read
            request(slot, ks);
        }
        rgmma::cp_async_wait<0>();
        __syncthreads();                                            // the tile is there; with two stages the last one is read
        if (stages == 2 && step + 1 < n_tiles) request(slot ^ 1, kv0 + (slot ^ 1) * stage);
        float sc[2][4] = {};
#pragma unroll 4
        for (int c = 0; c < d; c += 4) {
            float4 q4[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) q4[i] = *reinterpret_cast<const float4*>(qs + (2 * qa + i) * ld + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 k4 = *reinterpret_cast<const float4*>(ks + (ka + 16 * j) * ld + c);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    sc[i][j] += q4[i].x * k4.x; sc[i][j] += q4[i].y * k4.y;
                    sc[i][j] += q4[i].z * k4.z; sc[i][j] += q4[i].w * k4.w;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = ka + 16 * j;
                if (e >= n || 2 * qa + i >= nq) sc[i][j] = -INFINITY;
                else if (e0 + e >= w.x.start && !node_seen(a, w.x.row0 + (q0 + 2 * qa + i) / group, e0 + e - w.x.start)) sc[i][j] = -INFINITY;
                mx = fmaxf(mx, sc[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn, f = exp2f(m[i] - ms);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(sc[i][j] - ms);
                ps[(2 * qa + i) * TG_LD + ka + 16 * j] = p;
                sum += p;
            }
            l[i] = l[i] * f + sum;                                  // this thread's entries; added up at the end
            m[i] = mn;
            if (ka == 0) al[2 * qa + i] = f;
        }
        __syncthreads();
        look_up(slot);                                              // two tiles on: this one's rows are on their way since before the last barrier
#pragma unroll
        for (int i = 0; i < TG_Q; ++i) {
            const float f = al[i];
#pragma unroll
            for (int c = 0; c < COLS; ++c) acc[c][i] *= f;
        }
        const int some = (n + 4 * GROUPS - 1) / (4 * GROUPS) * (4 * GROUPS);   // the tile's rows up to 64 are zeros behind n
        for (int e = 4 * part; e < some; e += 4 * GROUPS) {
            float v[COLS][4];
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[c][j] = col + DP * c < d ? vs[(e + j) * ld + col + DP * c] : 0.f;
#pragma unroll
            for (int i = 0; i < TG_Q; ++i) {
                const float4 p4 = *reinterpret_cast<const float4*>(ps + i * TG_LD + e);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    acc[c][i] += p4.x * v[c][0]; acc[c][i] += p4.y * v[c][1];
                    acc[c][i] += p4.z * v[c][2]; acc[c][i] += p4.w * v[c][3];
                }
            }
        }
        if (!WHOLE && (step + 1 == n_tiles || w.last_tile())) {        // the item, or the stretch, ends: leave the part
            float sums[2] = {l[0], l[1]};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], o);
            }
            const size_t place = (size_t)w.first_query(a) + (size_t)blockIdx.x * TG_Q;
            if constexpr (GROUPS > 1) {                             // the groups' sums, added in their order, through this stage
                __syncthreads();
#pragma unroll
                for (int i = 0; i < TG_Q; ++i) ks[i * TG_THREADS + tid] = acc[0][i];
                __syncthreads();
                if (part == 0) {
#pragma unroll
                    for (int i = 0; i < TG_Q; ++i)
                        for (int g = 1; g < GROUPS; ++g) acc[0][i] += ks[i * TG_THREADS + g * DP + col];
                }
            }
            if (part == 0) {
#pragma unroll
                for (int i = 0; i < TG_Q; ++i)
                    if (i < nq)
#pragma unroll
                        for (int c = 0; c < COLS; ++c)
                            if (col + DP * c < d) a.part_o[(place + i) * d + col + DP * c] = acc[c][i];
            }
            if (ka == 0)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (2 * qa + i < nq) {
                        *reinterpret_cast<float2*>(a.part_ml + (place + 2 * qa + i) * 2) = make_float2(m[i], sums[i]);
                        const int qi = q0 + 2 * qa + i;
                        if (parts) a.parts[(size_t)(w.x.row0 + qi / group) * a.nh + w.kvh() * group + qi % group] = make_int2((int)place + 2 * qa + i, parts);
                    }
            __syncthreads();                                        // the queries, and what went through the tile, are read
        }
        if constexpr (WHOLE) ++w.tile;
        else w.next(a, step + 1 < n_tiles);
    }
    if constexpr (WHOLE) {
        __shared__ float fin_ml[TG_Q][2], row_ml[TG_Q][2];          // this block's M and L; the query's M and 1 / L
        cg::cluster_group cluster = cg::this_cluster();
        float* fin = kv0;                                           // [16][d]
        rgmma::cp_async_wait<0>();                                  // (where there was no tile, none was waited for)
        __syncthreads();                                            // the last tile is read
        if constexpr (GROUPS > 1) {                                 // the groups' sums, added in their order, behind what is left
            float* sums = kv0 + TG_Q * d;
#pragma unroll
            for (int i = 0; i < TG_Q; ++i) sums[i * TG_THREADS + tid] = acc[0][i];
            __syncthreads();
            if (part == 0) {
#pragma unroll
                for (int i = 0; i < TG_Q; ++i)
                    for (int g = 1; g < GROUPS; ++g) acc[0][i] += sums[i * TG_THREADS + g * DP + col];
            }
        }
        if (part == 0) {
#pragma unroll
            for (int i = 0; i < TG_Q; ++i)
                if (i < nq)
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
                        if (col + DP * c < d) fin[i * d + col + DP * c] = acc[c][i];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
            if (ka == 0) { fin_ml[2 * qa + i][0] = m[i]; fin_ml[2 * qa + i][1] = l[i]; }
        }
        cluster.sync();                                             // every block's result is in place
        if (tid < nq) join_cluster_ml(cluster, &fin_ml[0][0], tid, row_ml[tid][0], row_ml[tid][1]);
        __syncthreads();
        const int h0 = w.kvh() * group;
        // a warp has whole queries, so that it can work out again what is no number
        for (int i = rank * (TG_THREADS / 32) + (tid >> 5); i < nq; i += C * (TG_THREADS / 32)) {
            const int t = w.x.row0 + (q0 + i) / group, h = h0 + (q0 + i) % group;
            A* to = out + (size_t)t * out_ld + (size_t)h * d;
            bool odd = false;
            for (int c = tid & 31; c < d; c += 32) {
                float sum = 0.f;
                for (int k = 0; k < C; ++k)
                    sum += exp2f(cluster.map_shared_rank(&fin_ml[0][0], k)[i * 2] - row_ml[i][0]) * cluster.map_shared_rank(fin, k)[i * d + c];
                sum *= row_ml[i][1];
                odd |= !isfinite(sum);
                to[c] = from_f32<A>(sum);
            }
            if (__any_sync(0xffffffffu, odd)) row_by_formula<A>(a, w.x, w.r, t, h, to, 0, d);
        }
        cluster.sync();                                             // nobody leaves while its results are being read
    }
}

// ---------------------------------------------------------------------------------------------------
// Joining the parts of a row and head.
// ---------------------------------------------------------------------------------------------------
#define JOIN_THREADS 256

// A thread has four columns of a row and head: PS threads share their parts where there are few rows, and a thread has ITEMS of them where
// there are many, so that the blocks are resident at once (a block is there for two trips to memory, where the parts are and the parts
// themselves: 16 nodes of 64 requests, 2,056 blocks of one quad a thread, 16 us; 13 with two, 17 with four).
template <typename A, int PS, int ITEMS>
__global__ void __launch_bounds__(JOIN_THREADS) tree_join_kernel(const TreeArgs a, A* __restrict__ out, int out_ld) {
    constexpr int COLS = JOIN_THREADS / PS;                         // threads of a share
    __shared__ float4 s_acc[PS > 1 ? JOIN_THREADS : 1];
    __shared__ float2 s_ml[PS > 1 ? JOIN_THREADS : 1];
    pdl_wait();
    pdl_trigger();
    const unsigned d = a.d, quads = (d + 3) / 4, share = threadIdx.x / COLS, rows = (unsigned)a.T * a.nh;    // row: t x nh + h
    const size_t next = a.item_queries;
    const float2* mls = reinterpret_cast<const float2*>(a.part_ml);
    unsigned row[ITEMS], c[ITEMS];
    int n[ITEMS], place[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const unsigned item = (blockIdx.x * ITEMS + k) * COLS + threadIdx.x % COLS;
        row[k] = item / quads;
        c[k] = 4 * (item - row[k] * quads);
        const int2 where = row[k] < rows ? a.parts[row[k]] : make_int2(0, -1);
        // (of rows in no order at all nobody may have said: nothing outside is read)
        const bool mine = where.y >= 0 && where.x >= 0 && (long long)where.x + ((long long)where.y - 1) * a.item_queries < a.places;
        place[k] = mine ? where.x : 0;
        n[k] = mine ? where.y : -1;
    }
    float M[ITEMS], L[ITEMS];
    float4 acc[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        M[k] = -INFINITY;
        L[k] = 0.f;
        acc[k] = {0.f, 0.f, 0.f, 0.f};
    }
    constexpr int AHEAD = ITEMS > 1 ? 2 : 4;                        // parts that are asked for together
    auto some = [&](int k, int i) {                                 // parts i, i + PS, ... of item k
        float2 ml[AHEAD];
        float4 y[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            ml[j] = make_float2(-INFINITY, 0.f);
            y[j] = {0.f, 0.f, 0.f, 0.f};
            if (i + j * PS < n[k]) {
                const size_t at = place[k] + (size_t)(i + j * PS) * next;
                const float* from = a.part_o + at * d + c[k];
                ml[j] = mls[at];
                if (d % 4 == 0) y[j] = *reinterpret_cast<const float4*>(from);
                else { y[j].x = from[0]; if (c[k] + 1 < d) y[j].y = from[1]; if (c[k] + 2 < d) y[j].z = from[2]; if (c[k] + 3 < d) y[j].w = from[3]; }
            }
        }
        float m = M[k];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) m = fmaxf(m, ml[j].x);
        const float ms = m == -INFINITY ? 0.f : m, f = exp2f(M[k] - ms);
        L[k] *= f; acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const float fj = exp2f(ml[j].x - ms);
            L[k] += fj * ml[j].y;
            acc[k].x += fj * y[j].x; acc[k].y += fj * y[j].y; acc[k].z += fj * y[j].z; acc[k].w += fj * y[j].w;
        }
        M[k] = m;
    };
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) some(k, (int)share);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        for (int i = (int)share + AHEAD * PS; i < n[k]; i += AHEAD * PS) some(k, i);
    if constexpr (PS > 1) {                                         // the shares, in their order (one item a thread)
        s_acc[threadIdx.x] = acc[0];
        s_ml[threadIdx.x] = make_float2(M[0], L[0]);
        __syncthreads();
        if (share == 0) {
            float m = M[0];
#pragma unroll
            for (int k = 1; k < PS; ++k) m = fmaxf(m, s_ml[threadIdx.x + k * COLS].x);
            const float ms = m == -INFINITY ? 0.f : m;
            L[0] = 0.f;
            acc[0] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < PS; ++k) {
                const float2 ml = s_ml[threadIdx.x + k * COLS];
                const float4 y = s_acc[threadIdx.x + k * COLS];
                const float f = exp2f(ml.x - ms);
                L[0] += f * ml.y;
                acc[0].x += f * y.x; acc[0].y += f * y.y; acc[0].z += f * y.z; acc[0].w += f * y.w;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        bool odd = false;
        if (n[k] >= 0 && share == 0) {
            const float inv = L[k] == 0.f ? 0.f : 1.f / L[k];
            const float4 v = {acc[k].x * inv, acc[k].y * inv, acc[k].z * inv, acc[k].w * inv};
            odd = !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w));
            const unsigned t = row[k] / a.nh, h = row[k] - t * a.nh;
            A* to = out + (size_t)t * out_ld + (size_t)h * d + c[k];
            if (sizeof(A) == 2 && c[k] + 3 < d && ((uintptr_t)to & 7) == 0) {
                *reinterpret_cast<uint2*>(to) = make_uint2(rgmma::pack_bf16(v.x, v.y), rgmma::pack_bf16(v.z, v.w));
            } else {
                to[0] = from_f32<A>(v.x);
                if (c[k] + 1 < d) to[1] = from_f32<A>(v.y);
                if (c[k] + 2 < d) to[2] = from_f32<A>(v.z);
                if (c[k] + 3 < d) to[3] = from_f32<A>(v.w);
            }
        }
        // Columns that are no numbers: the warp works them out again, from the first such column of a row and head to the last that it has.
        for (unsigned left = __ballot_sync(0xffffffffu, odd); left;) {
            const unsigned i = __shfl_sync(0xffffffffu, row[k], __ffs(left) - 1), same = __ballot_sync(0xffffffffu, odd && row[k] == i);
            const int from = __shfl_sync(0xffffffffu, c[k], __ffs(same) - 1), last = __shfl_sync(0xffffffffu, c[k], 31 - __clz(same));
            const int t = i / a.nh, h = i % a.nh, r = request_of(a, t);
            if (r >= 0) row_by_formula<A>(a, tree_request(a, r), r, t, h, out + (size_t)t * out_ld + (size_t)h * d, from, min(a.d, last + 4));
            left &= ~same;
        }
    }
}

// ---------------------------------------------------------------------------------------------------
static size_t tg_smem(int d) { return (size_t)(TG_Q * tg_row(d) + tg_stages(d) * tg_stage(d) + TG_Q * TG_LD + TG_Q) * sizeof(float); }

// cluster: not 0, an item to a cluster of so many blocks.
static int launch_tree_general(const TreeArgs& a, int dtype, void* out, int out_ld, int cluster, int q_blocks, cudaStream_t s) {
    const size_t smem = tg_smem(a.d);
    const bool vec = a.d % 4 == 0 && (((uintptr_t)a.kv) & (dtype == RG_DTYPE_F32 ? 15 : 7)) == 0;
    const long long blocks = cluster ? (long long)a.R * a.nkv * q_blocks * cluster : a.workers;
    if (blocks > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
#define RG_TG_(A, DP, VEC, W) { RG_ALLOW_SMEM((tree_general_kernel<A, DP, VEC, W>), 160 * 1024) \
    return rg_launch(tree_general_kernel<A, DP, VEC, W>, dim3((unsigned)blocks), dim3(TG_THREADS), smem, s, cluster, a, (A*)out, out_ld, q_blocks); }
#define RG_TG(A, DP, VEC) { if (cluster) RG_TG_(A, DP, VEC, true) RG_TG_(A, DP, VEC, false) }
#define RG_TG_WIDTH(A, VEC) { if (a.d <= 32) RG_TG(A, 32, VEC) if (a.d <= 64) RG_TG(A, 64, VEC) RG_TG(A, 128, VEC) }
    if (dtype == RG_DTYPE_F32) { if (vec) RG_TG_WIDTH(float, true) RG_TG_WIDTH(float, false) }
    if (vec) RG_TG_WIDTH(bf16, true)
    RG_TG_WIDTH(bf16, false)
#undef RG_TG_WIDTH
#undef RG_TG
#undef RG_TG_
}

// See attention_tree.cuh for the arguments.  Scratch: part_o [T nh + workers item_queries, d] on a boundary of 32 bytes, part_ml [.., 2] and
// parts [T, nh] on one of 8.  tensor_cores: 0 tree_general_kernel; 1 tree_tc_kernel, a stretch a side; 2 the same,
// a stretch for both sides; tile_rows: rows of a side.  cluster: not 0, items of 16 queries to clusters of so many blocks, in one launch and
// without scratch.
extern "C" int rg_tree_attention(const void* q, int q_stride, void* out, int out_ld, const void* kv, int num_pages, int dtype,
                                 const int* block_table, int max_blocks, const int* cu_rows, const int* starts, const int* masks, int words,
                                 int R, int T, int nh, int nkv, int d, int page_size, float scale, int max_rows, int max_context,
                                 int blocks, int workers, int item_queries, int least, int tile_rows, int tensor_cores, int cluster, float* part_o, float* part_ml,
                                 int2* parts, int* err, void* stream) {
    if (T <= 0 || R <= 0 || max_rows <= 0) return 0;
    if (d < 1 || d > 256 || num_pages < 1 || nkv < 1 || nh < nkv || nh % nkv || page_size < 1 || max_blocks < 0 || words < 0 || max_context < 0 || out_ld < nh * d ||
        (!cluster && workers < 1) || item_queries < 1 || least < 1 || ((uintptr_t)part_o & 31) || ((uintptr_t)part_ml & 7) || ((uintptr_t)parts & 7) ||
        (long long)T * nh + (long long)workers * item_queries > 0x7fffffffll)
        return RG_ERR_UNSUPPORTED;
    TreeArgs a = {};
    a.q = q; a.q_stride = q_stride; a.kv = kv; a.block_table = block_table; a.max_blocks = max_blocks; a.cu_rows = cu_rows; a.starts = starts;
    a.masks = masks; a.words = words; a.R = R; a.T = T; a.nh = nh; a.nkv = nkv; a.d = d; a.page_size = page_size; a.pages = num_pages;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.max_rows = max_rows;
    a.limit = (int)min((long long)max_context, min(0x7fffff00ll, (long long)max_blocks * page_size));
    a.workers = workers; a.item_queries = item_queries; a.least = least;
    a.part_o = part_o; a.part_ml = part_ml; a.parts = parts; a.err = err;
    a.places = T * nh + workers * item_queries;
    a.page_shift = -1;
    for (int b = 0; b < 31; ++b) if (page_size == (1 << b)) a.page_shift = b;
    a.tile = tensor_cores ? TT_STAGE : TG_K;
    a.begin = tensor_cores ? TT_BEGIN : TG_BEGIN;
    if (cluster) {
        if (cluster > 8 || tensor_cores || item_queries != TG_Q) return RG_ERR_UNSUPPORTED;
        const long long q_blocks = ((long long)max_rows * (nh / nkv) + TG_Q - 1) / TG_Q;
        if (q_blocks * nkv * R * cluster > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
        if (tree_rows_ok(a, dtype)) return launch_tree_rows(a, (bf16*)out, out_ld, cluster, (int)q_blocks, (cudaStream_t)stream);
        return launch_tree_general(a, dtype, out, out_ld, cluster, (int)q_blocks, (cudaStream_t)stream);
    }
    if (tensor_cores ? !tree_tc_ok(a, dtype) : item_queries != TG_Q || workers != blocks) return RG_ERR_UNSUPPORTED;
    int e = tensor_cores ? launch_tree_tc(a, tile_rows, tensor_cores == 2, blocks, (cudaStream_t)stream) : launch_tree_general(a, dtype, out, out_ld, 0, 0, (cudaStream_t)stream);
    if (e) return e;
    const long long threads = (long long)T * nh * ((d + 3) / 4), joins = (threads + JOIN_THREADS - 1) / JOIN_THREADS;
    if (threads > 0x7fff0000ll) return RG_ERR_UNSUPPORTED;
#define RG_TJ(A, PS, ITEMS) return rg_launch(tree_join_kernel<A, PS, ITEMS>, dim3((unsigned)((threads * PS + JOIN_THREADS * ITEMS - 1) / (JOIN_THREADS * ITEMS))), \
                                             dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a, (A*)out, out_ld);
#define RG_TJ_SHARES(A) { if (joins > 592) RG_TJ(A, 1, 2) if (joins > 148) RG_TJ(A, 1, 1) RG_TJ(A, 4, 1) }
    if (dtype == RG_DTYPE_F32) RG_TJ_SHARES(float)
    RG_TJ_SHARES(bf16)
#undef RG_TJ_SHARES
#undef RG_TJ
}
