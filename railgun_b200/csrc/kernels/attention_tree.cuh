// What the kernels of attention_tree.cu share: how the work of trees of drafted tokens is cut, and where the parts are left.
//
// Request r brings rows cu_rows[r] .. cu_rows[r + 1] - 1, the nodes of its tree, behind starts[r] entries that it has in the
// cache; node j is entry starts[r] + j.  Row i sees the entries before starts[r] and the nodes whose bit its mask has:
//   out_ih = sum_e p_ih(e) v_e,  p = softmax over {e < start} and {start + j : bit j of mask i} of scale q_ih . k_e,   no entry: 0
//
// An item is (request, kv head, block of queries); query i of a request and kv head is row i / group, head i % group.  An item has
// ceil(entries / tile) tiles.  All items' tiles, one item after the other, are one line that is cut into as many stretches of `per`
// tiles as there are workers: whatever the requests' lengths, every worker has the same number of tiles to read.  A stretch
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
    int tile, item_queries, workers, least;     // entries of a tile, queries of an item, workers, least tiles of a stretch
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
    x.blocks = (int)(((long long)x.rows * (a.nh / a.nkv) + a.item_queries - 1) / a.item_queries);
    return x;
}
__device__ __forceinline__ long long tree_tiles(const TreeArgs& a, const TreeRequest& x) { return (long long)x.tiles * x.blocks * a.nkv; }

// Tiles of all items, and where (up to two) workers begin: a request, -1: nowhere, and a place among its tiles.
struct TreeStart {
    long long total, per;
    long long in[2];
    int r[2];
    TreeRequest x[2];
};

// Where a worker is on the line: an item and a tile of it.
struct TreeWalk {
    TreeRequest x;
    int r, item, tile;           // item: kv head x blocks + block of queries
    __device__ __forceinline__ int kvh() const { return item / x.blocks; }
    __device__ __forceinline__ int block() const { return item % x.blocks; }
    __device__ __forceinline__ void skip_empty(const TreeArgs& a) {      // to a request that has tiles (one is known to come)
        while (x.tiles == 0 || x.blocks == 0) x = tree_request(a, ++r);
    }
    // Where worker i of `st` begins.
    __device__ __forceinline__ void at(const TreeStart& st, int i) {
        r = st.r[i];
        x = st.x[i];
        const long long in = st.in[i];
        item = in >> 32 ? (int)(in / x.tiles) : (int)((unsigned)in / (unsigned)x.tiles);
        tile = (int)(in - (long long)item * x.tiles);
    }
    // One tile on; `more`: there is one.
    __device__ __forceinline__ void next(const TreeArgs& a, bool more) {
        if (++tile < x.tiles) return;
        tile = 0;
        if (++item < x.blocks * a.nkv) return;
        item = 0;
        if (!more) return;
        x = tree_request(a, ++r);
        skip_empty(a);
    }
    __device__ __forceinline__ bool last_tile() const { return tile + 1 == x.tiles; }
    // In how many parts the item is cut whose first tile is a worker's `done`-th.
    __device__ __forceinline__ int parts(int done, long long per) const { return (int)((unsigned)(done + x.tiles - 1) / (unsigned)min(per, 0x7fffffffll)) + 1; }
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

// The whole block, THREADS threads: tiles of all items, and the request (with the place among its tiles) in which each of `n`
// (up to 2) workers, `first` and `first` + `apart`, begins (r -1: it has nothing).  The last block says which rows nobody has.
template <int THREADS>
__device__ __forceinline__ void tree_plan(const TreeArgs& a, int first, int n, int apart, TreeStart& st) {
    __shared__ long long sums[THREADS / 32 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](long long v, long long& total) -> long long {       // exclusive, over the block
        long long x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = x;
        __syncthreads();
        long long before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        return before + x - v;
    };
    long long total = 0, mine = 0, before = 0;
    TreeRequest x;
    if (threadIdx.x < 2) st.r[threadIdx.x] = -1;
    for (int r0 = 0; r0 < a.R; r0 += THREADS) {
        const int r = r0 + threadIdx.x;
        long long some;
        if (r < a.R) x = tree_request(a, r);
        mine = r < a.R ? tree_tiles(a, x) : 0;
        before = total + scan(mine, some);
        total += some;
    }
    const long long per = max((long long)a.least, total >> 31 ? (total + a.workers - 1) / a.workers : (long long)((unsigned)total + a.workers - 1u) / a.workers);
    if (threadIdx.x == 0) {
        st.total = total;
        st.per = per;
    }
    const bool once = a.R <= THREADS;                                    // what was found above still stands
    long long sofar = 0;
    for (int r0 = 0; r0 < a.R; r0 += THREADS) {
        const int r = r0 + threadIdx.x;
        if (!once) {
            long long some;
            if (r < a.R) x = tree_request(a, r);
            mine = r < a.R ? tree_tiles(a, x) : 0;
            before = sofar + scan(mine, some);
            sofar += some;
        }
        if (r >= a.R) continue;
        for (int i = 0; i < n; ++i) {
            const long long at = (first + (long long)i * apart) * per - before;
            if (at >= 0 && at < mine) { st.r[i] = r; st.in[i] = at; st.x[i] = x; }
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
