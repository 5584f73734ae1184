// What the kernels of attention_tree.cu share: how the work of trees of drafted tokens is cut, and where the parts are left.
//
// Request r brings rows cu_rows[r] .. cu_rows[r + 1] - 1, the nodes of its tree, behind starts[r] entries that it has in the
// cache; node j is entry starts[r] + j.  Row i sees the entries before starts[r] and the nodes whose bit its mask has:
//   out_ih = sum_e p_ih(e) v_e,  p = softmax over {e < start} and {start + j : bit j of mask i} of scale q_ih . k_e,   no entry: 0
//
// An item is (request, kv head, block of queries); query i of a request and kv head is row i / group, head i % group.  An item has
// ceil(entries / tile) tiles.  All items' tiles, one item after the other, are one line that is cut into as many stretches of `per`
// places as there are workers: whatever the requests' lengths, every worker has the same work.  In front of an item's tiles are `begin`
// places that hold none, for what an item costs a worker besides (the last one's part left, queries and a first maximum had).  A stretch
// may end inside an item; what a worker finds for an item, its part, is left as the unnormalised output o = sum 2^(s - m) v with
// m = max s and l = sum 2^(s - m), s = scale log2(e) q.k, in 32-bit, and a second kernel joins the parts of every row and head:
//   out = sum_parts 2^(m - M) o / sum_parts 2^(m - M) l,   M = max_parts m
// A part's numbers lie at (first query of the item in all queries) + worker x (queries of an item): parts along the line never
// meet, and T x nh + workers x (queries of an item) places are enough.  Who finds an item's first part also says where it is and how
// many there are, so that the kernel that joins takes two trips to memory: with the requests looked up and the line worked out again
// there, 16 nodes of 64 requests (32 heads of 128) took 25 us to join, 13 so.
#pragma once
#include "common.cuh"

#define RG_BAD_PAGE 1000              // in the error flag: a table names a page that the cache does not have

struct TreeArgs {
    const void* q;               // [T, q_stride]: head h of row t at q[t * q_stride + h * d]
    const void* kv;              // [pages, 2, nkv, page_size, d]
    const int* block_table;      // [R, max_blocks]
    const int* cu_rows;          // [R + 1]
    const int* starts;           // [R]
    const int* masks;            // [T, words]
    float* part_o;               // [places, d]
    float* part_ml;              // [places, 2]
    int2* parts;                 // [T, nh]: where a row and head's first part is, and how many there are (-1: a row that is left as it was)
    int places;                  // of parts
    int* err;
    int R, T, max_rows, limit;   // limit: the most entries of a request that are seen
    int q_stride, max_blocks, words, pages;
    int nh, nkv, d, page_size, page_shift;      // page_shift: log2 of the page size, or -1
    int tile, item_queries, workers, least;     // entries of a tile, queries of an item, workers, least places of a stretch
    int begin;                   // places in front of an item's tiles
    float scale_log2;
};

// A request as the kernels see it: rows that take part, entries that are seen, tiles of an item and items of a kv head.
struct TreeRequest {
    int row0, rows, start, entries, tiles, blocks;
};
__device__ __forceinline__ TreeRequest tree_request(const TreeArgs& a, int r) {
    TreeRequest x;
    const int row0 = a.cu_rows[r], next = a.cu_rows[r + 1], start = a.starts[r];
    x.row0 = row0;
    const long long rows = min((long long)next - row0, (long long)a.max_rows);
    x.rows = row0 < 0 || start < 0 ? 0 : (int)max(0ll, min(rows, (long long)a.T - row0));
    x.start = start;
    x.entries = x.rows ? (int)min((long long)a.limit, (long long)start + x.rows) : 0;
    x.tiles = (x.entries + a.tile - 1) / a.tile;
    x.blocks = (int)(((unsigned)x.rows * (unsigned)(a.nh / a.nkv) + a.item_queries - 1u) / (unsigned)a.item_queries);   // (T x nh is below 2^31)
    return x;
}
// Places of a stretch, and of up to two workers: where they begin (a request, -1: nowhere; an item of it; a place of that) and how many
// tiles lie on the line before that and before their end.
struct TreeStart {
    long long per, from[2], to[2];
    int r[2], item[2], in[2];
    TreeRequest x[2];
    __device__ __forceinline__ int tiles(int i) const { return r[i] < 0 ? 0 : (int)min(0x7fffffffll, to[i] - from[i]); }
};

// Where a worker is on the line: an item and a tile of it.
struct TreeWalk {
    TreeRequest x;
    int r, item, tile;           // item: kv head x blocks + block of queries
    int place;                   // of the tile, in the worker's stretch
    __device__ __forceinline__ int kvh() const { return item / x.blocks; }
    __device__ __forceinline__ int block() const { return item % x.blocks; }
    __device__ __forceinline__ void skip_empty(const TreeArgs& a) {      // to a request that has tiles (one is known to come)
        while (x.tiles == 0 || x.blocks == 0) x = tree_request(a, ++r);
    }
    // The first tile of worker i of `st`, which has some.
    __device__ __forceinline__ void at(const TreeArgs& a, const TreeStart& st, int i) {
        r = st.r[i];
        x = st.x[i];
        item = st.item[i];
        place = max(0, a.begin - st.in[i]);
        tile = max(0, st.in[i] - a.begin);
    }
    // n tiles on, of which all but the last are this item's; `more`: there is one.
    __device__ __forceinline__ void next(const TreeArgs& a, bool more, int n = 1) {
        place += n;
        if ((tile += n) < x.tiles) return;
        tile = 0;
        place += a.begin;
        if (++item < x.blocks * a.nkv) return;
        item = 0;
        if (!more) return;
        x = tree_request(a, ++r);
        skip_empty(a);
    }
    __device__ __forceinline__ bool last_tile() const { return tile + 1 == x.tiles; }
    // In how many parts the item is cut whose first tile this is.
    __device__ __forceinline__ int parts(long long per) const {
        return (int)((unsigned)(place + x.tiles - 1) / (unsigned)min(per, 0x7fffffffll)) + 1;
    }
    // The first query of the item among all rows' and heads'.
    __device__ __forceinline__ long long first_query(const TreeArgs& a) const {
        return (long long)x.row0 * a.nh + (long long)kvh() * x.rows * (a.nh / a.nkv) + (long long)block() * a.item_queries;
    }
};

// Rows that no request has, or that no launch was sized for, have no parts and are left as they were; rows without entries have none and
// become 0.
template <int THREADS>
__device__ __forceinline__ void tree_gaps(const TreeArgs& a) {
    auto say = [&](int t, int n) {
        for (int h = 0; h < a.nh; ++h) a.parts[(size_t)t * a.nh + h] = make_int2(0, n);
    };
    const int begin = max(0, min(a.cu_rows[0], a.T)), end = max(0, min(a.cu_rows[a.R], a.T));
    for (size_t i = threadIdx.x; i < (size_t)begin * a.nh; i += THREADS) a.parts[i] = make_int2(0, -1);
    for (size_t i = (size_t)end * a.nh + threadIdx.x; i < (size_t)a.T * a.nh; i += THREADS) a.parts[i] = make_int2(0, -1);
    for (int r = threadIdx.x; r < a.R; r += THREADS) {
        const TreeRequest x = tree_request(a, r);
        const int next = min(a.cu_rows[r + 1], a.T);
        if (x.row0 < 0) continue;
        for (int t = x.row0 + x.rows; t < next; ++t) say(t, -1);
        if (x.tiles == 0)
            for (int t = x.row0; t < x.row0 + x.rows; ++t) say(t, 0);
    }
}

// The whole block, THREADS threads: where each of `n` (up to 2) workers, `first` and `first` + `apart`, begins and how many tiles it
// has.  The last block says which rows nobody has.
template <int THREADS>
__device__ __forceinline__ void tree_plan(const TreeArgs& a, int first, int n, int apart, TreeStart& st) {
    __shared__ long long s_places[THREADS / 32];
    __shared__ int s_items[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // Loops stay loops here: this code runs once a launch and comes from memory, each 128 bytes of it a trip.
    long long mine = 0, before = 0, total = 0;                           // places of this thread's request, of the requests before it, of all
    int items = 0, items_before = 0, items_total = 0;
    TreeRequest x;
    auto look = [&](int r0) {                                            // at THREADS requests from r0 on; what came before is in the totals
        const int r = r0 + threadIdx.x, some = a.R - r0;
        items = 0;
        mine = 0;
        if (r < a.R) {
            x = tree_request(a, r);
            items = x.tiles ? x.blocks * a.nkv : 0;
            mine = (long long)items * (x.tiles + a.begin);
        }
        long long p = mine;
        int n = items;
#pragma unroll 1
        for (int o = 1; o < 32; o <<= 1) {
            const long long q = __shfl_up_sync(0xffffffffu, p, o);
            const int m = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) { p += q; n += m; }
        }
        __syncthreads();
        if (lane == 31) { s_places[warp] = p; s_items[warp] = n; }
        __syncthreads();
        before = total + p - mine;
        items_before = items_total + n - items;
#pragma unroll 1
        for (int w = 0; w < THREADS / 32 && 32 * w < some; ++w) {
            if (w < warp) { before += s_places[w]; items_before += s_items[w]; }
            total += s_places[w];
            items_total += s_items[w];
        }
    };
    if (threadIdx.x < 2) st.r[threadIdx.x] = -1;
    for (int r0 = 0; r0 < a.R; r0 += THREADS) look(r0);
    const long long all = total;
    const long long per = max((long long)a.least, all >> 31 ? (all + a.workers - 1) / a.workers : (long long)(((unsigned)all + a.workers - 1u) / a.workers));
    if (threadIdx.x == 0) st.per = per;
    if (threadIdx.x < n && (first + (long long)threadIdx.x * apart + 1) * per >= all) st.to[threadIdx.x] = all - (long long)items_total * a.begin;
    const bool once = a.R <= THREADS;                                    // what was found above still stands
    if (!once) total = items_total = 0;
    for (int r0 = 0; r0 < a.R; r0 += THREADS) {
        if (!once) look(r0);
        if (mine == 0) continue;
        const int len = x.tiles + a.begin;
#pragma unroll 1
        for (int i = 0; i < 2 * n; ++i) {                                // the places where the workers begin, and where they end
            const long long place = (first + (long long)(i >> 1) * apart + (i & 1)) * per, at = place - before;
            if (at < 0 || at >= mine) continue;
            const int item = at >> 32 ? (int)(at / len) : (int)((unsigned)at / (unsigned)len), in = (int)(at - (long long)item * len);
            const long long tiles = place - (long long)(items_before + item) * a.begin - min(in, a.begin);
            if (i & 1) st.to[i >> 1] = tiles;
            else {
                st.from[i >> 1] = tiles;
                st.r[i >> 1] = r0 + threadIdx.x;
                st.item[i >> 1] = item;
                st.in[i >> 1] = in;
                st.x[i >> 1] = x;
            }
        }
    }
    if (blockIdx.x == gridDim.x - 1) tree_gaps<THREADS>(a);
    __syncthreads();
}

__device__ __forceinline__ bool node_seen(const TreeArgs& a, int row, int node) {
    return (node >> 5) < a.words && (a.masks[(size_t)row * a.words + (node >> 5)] >> (node & 31) & 1);
}
// Where entry e of request r is in the cache (its key of kv head kvh); a page that the cache does not have is reported, and read
// as its first one.
__device__ __forceinline__ long long entry_at(const TreeArgs& a, int r, int kvh, int e) {
    int page = a.block_table[(size_t)r * a.max_blocks + e / a.page_size];
    if ((unsigned)page >= (unsigned)a.pages) { atomicCAS(a.err, 0, RG_BAD_PAGE); page = 0; }
    return (((long long)page * 2 * a.nkv + kvh) * a.page_size + e % a.page_size) * a.d;
}

// Row t's request (-1: none that has it among its rows).  Whole warps, all lanes for the same row: a lane looks at every 32nd.
__device__ __forceinline__ int request_of(const TreeArgs& a, int t) {
    const int lane = threadIdx.x & 31;
    unsigned hit = 0;
    int r0 = 0;
#pragma unroll 1
    for (; !hit && r0 < a.R; r0 += 32) {
        const int r = min(r0 + lane, a.R - 1), first = a.cu_rows[r], next = a.cu_rows[r + 1];
        hit = __ballot_sync(0xffffffffu, r0 + lane < a.R && first >= 0 && t >= first && t < next);
    }
    return hit ? r0 - 32 + __ffs(hit) - 1 : -1;
}

// Row t, head h as the formula has it, by one warp, from the cache: entry by entry, and an entry that is not seen is not read into a
// sum; columns from_col .. to_col - 1 are written.  For rows whose output is no number or infinite: 0, the weight of an entry that is not seen, times such a value is no number.
template <typename A>
__device__ __noinline__ void row_by_formula(const TreeArgs& a, const TreeRequest& x, int r, int t, int h, A* to, int from_col, int to_col) {
    const int lane = threadIdx.x & 31, d = a.d, group = a.nh / a.nkv, kvh = h / group;
    const A* q = (const A*)a.q + (size_t)t * a.q_stride + (size_t)h * d;
    const A* kv = (const A*)a.kv;
    const size_t to_values = (size_t)a.nkv * a.page_size * d;
    float M = -INFINITY, L = 0.f, acc[8] = {};                      // columns lane + 32 k
    for (int e0 = 0; e0 < x.entries; e0 += 32) {
        const int e = e0 + lane;
        const bool seen = e < x.entries && (e < x.start || node_seen(a, t, e - x.start));
        const long long at = seen ? entry_at(a, r, kvh, e) : 0;
        float s = -INFINITY;
        if (seen) {
            s = 0.f;
            for (int c = 0; c < d; ++c) s += to_f32(q[c]) * a.scale_log2 * to_f32(kv[at + c]);
        }
        if (__any_sync(0xffffffffu, seen && !(s < INFINITY))) {     // a score that is no number, or infinite: so is the whole row
            L = NAN;
            break;
        }
        const float mn = fmaxf(M, warp_max(s)), ms = mn == -INFINITY ? 0.f : mn, f = exp2f(M - ms), p = exp2f(s - ms);
        L = L * f + warp_sum(p);
        M = mn;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] *= f;
        for (unsigned left = __ballot_sync(0xffffffffu, seen); left; left &= left - 1) {
            const int j = __ffs(left) - 1;
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const long long vj = __shfl_sync(0xffffffffu, at, j) + (long long)to_values;
            if (pj == 0.f) continue;                                // a score of -infinity, or far below the others
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (lane + 32 * k < d) acc[k] += pj * to_f32(kv[vj + lane + 32 * k]);
        }
        bool settled = true;                                        // what is no number stays so
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (lane + 32 * k >= from_col && lane + 32 * k < to_col) settled &= acc[k] != acc[k];
        if (__all_sync(0xffffffffu, settled)) break;
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (lane + 32 * k >= from_col && lane + 32 * k < to_col) to[lane + 32 * k] = from_f32<A>(acc[k] * inv);
}

// Item number i of a launch with q_blocks blocks of queries for every request and kv head; false: the request has no such queries.
__device__ __forceinline__ bool tree_item(const TreeArgs& a, unsigned i, int q_blocks, TreeWalk& w) {
    const unsigned block = i % q_blocks, rk = i / q_blocks, kvh = rk % a.nkv;
    w.r = rk / a.nkv;
    w.x = tree_request(a, w.r);
    w.item = kvh * w.x.blocks + block;
    w.tile = 0;
    return block < w.x.blocks;
}
