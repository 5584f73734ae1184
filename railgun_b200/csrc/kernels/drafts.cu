// Trees of drafted tokens: their layout, and what is kept of them.
//
// Request r brings rows cu_rows[r] .. cu_rows[r + 1] - 1, the nodes of its tree: node 0 is the last token that is certain, another
// node continues its parent, which comes before it; parents[row] is its number within the request.  Node j is entry
// starts[r] + j of the request's cache.
#include "common.cuh"

#define RG_BAD_PAGE 1000               // in the error flag: a table names a page, or a request an entry, that the cache does not have
#define DRAFT_MOST 4096                // nodes of a tree

struct DraftRows {
    const int* cu_rows;          // [R + 1]
    const int* starts;           // [R]
    int R, T, max_rows;
};
// Request r's first row and how many rows it has (0: it is left out).
__device__ __forceinline__ int draft_rows(const DraftRows& d, int r, int& row0, int& start) {
    const int next = d.cu_rows[r + 1];
    row0 = d.cu_rows[r];
    start = d.starts[r];
    if (row0 < 0 || start < 0) return 0;
    return (int)max(0ll, min(min((long long)next - row0, (long long)d.max_rows), (long long)d.T - row0));
}

// ---------------------------------------------------------------------------------------------------
// Which nodes a node sees (itself and its ancestors, bit j of a row's mask for node j), and its position, start + how many
// ancestors it has.  Nodes go in groups of 32, a word of a mask each.  A warp has a group: five steps, in each of which a node
// takes over what the node sees that its line has been followed to, find the whole line inside the group and the first ancestor
// before it.  Then a thread goes up from its node, a group at a time: a word for each that the line touches, zeros for the others, every
// word written once.  A block has up to 256 rows of a request and looks at the groups up to its last; the last blocks write zeros for
// rows of no request.  Bound by the launch and two trips to memory: one tree of 16 nodes 1.8 us,
// 64 of up to 256 3.1 (one ancestor at a time 4.8), 12 chains of up to 343 3.0 (62), one of 4,096 31.
// ---------------------------------------------------------------------------------------------------
#define LAYOUT_THREADS 256
__global__ void __launch_bounds__(LAYOUT_THREADS) draft_tree_kernel(const DraftRows dr, const int* __restrict__ parents, int* __restrict__ masks,
                                                                    int words, int* __restrict__ positions) {
    extern __shared__ int2 line[];                                    // of a node: what it sees of its group, the first ancestor before that
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    auto nothing = [&](long long t) {
        for (int w = 0; w < words; ++w) masks[t * words + w] = 0;
        positions[t] = 0;
    };
    const long long mine = (long long)blockIdx.y * LAYOUT_THREADS + tid, every = (long long)gridDim.y * LAYOUT_THREADS;
    if (r == dr.R) {
        const int first = dr.R ? max(0, min(dr.cu_rows[0], dr.T)) : 0, end = dr.R ? max(0, min(dr.cu_rows[dr.R], dr.T)) : 0;
        for (long long t = mine; t < first; t += every) nothing(t);
        for (long long t = end + mine; t < dr.T; t += every) nothing(t);
        return;
    }
    int row0, start;
    const int n = draft_rows(dr, r, row0, start), last = min(n, ((int)blockIdx.y + 1) * LAYOUT_THREADS);
    if ((int)blockIdx.y * LAYOUT_THREADS < n) {
        for (int i0 = tid - lane; i0 < last; i0 += LAYOUT_THREADS) {
            const int i = i0 + lane;
            int before = i < n ? parents[row0 + i] : -1, to = lane;
            if (before >= i) before = -1;                             // no parent that comes before it: a root
            if (before >= i0) to = before - i0;
            unsigned bits = 1u << lane;
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                bits |= __shfl_sync(0xffffffffu, bits, to);
                to = __shfl_sync(0xffffffffu, to, to);
            }
            before = __shfl_sync(0xffffffffu, before, to);            // the line's first node in the group has its parent before it, or none
            line[i] = make_int2((int)bits, before);
        }
    }
    __syncthreads();
    if (mine < n) {
        int* mask = masks + (size_t)(row0 + mine) * words;
        int word = words - 1, node = (int)mine, depth = -1;
        while (node >= 0) {
            const int2 at = line[node];
            for (; word > node >> 5; --word) mask[word] = 0;
            mask[word--] = at.x;
            depth += __popc(at.x);
            node = at.y;
        }
        for (; word >= 0; --word) mask[word] = 0;
        positions[row0 + mine] = start + depth;
    }
    // rows beyond what the call says see nothing
    const long long all = min((long long)dr.cu_rows[r + 1], (long long)dr.T);
    if (row0 >= 0)
        for (long long t = row0 + n + mine; t < all; t += every) nothing(t);
}

extern "C" int rg_draft_tree(const int* parents, const int* cu_rows, const int* starts, int R, int T, int max_rows, int* masks, int words,
                             int* positions, void* stream) {
    if (T <= 0) return 0;
    if (R < 0 || max_rows < 0 || max_rows > DRAFT_MOST || words != (max_rows + 31) / 32) return RG_ERR_UNSUPPORTED;
    const DraftRows dr = {cu_rows, starts, R, T, max_rows};
    const int groups = (max_rows + LAYOUT_THREADS - 1) / LAYOUT_THREADS;
    return rg_launch(draft_tree_kernel, dim3((unsigned)R + 1, (unsigned)(groups ? groups : 1)), dim3(LAYOUT_THREADS), (size_t)words * 32 * sizeof(int2),
                     (cudaStream_t)stream, 1, dr, parents, masks, words, positions);
}

// ---------------------------------------------------------------------------------------------------
// The path of nodes that the model's own choices confirm: from node 0 on, the lowest child that holds the token chosen behind its
// parent.  Its entries move together behind the context in every cache: the k-th node's to entry start + k.  A path's nodes
// have rising numbers, so entry k is never the source of a later move: a thread takes some columns of a row of the cache and loads
// several moves' before it stores them, in their order, and no two threads touch the same columns.
// Every block works out the path of its request for itself (three numbers a node); the first one of a request writes the results.
// What bounds it is trips to memory one behind the other (rows, parents and tokens, choices, the table, entries there and back): one
// request of 16 nodes in 16 layers 4 us, 64 requests in 32 layers 10, of which the 33 MB that move are 5.
// ---------------------------------------------------------------------------------------------------
#define KEEP_THREADS 256
#define KEEP_AHEAD 8
#define KEEP_CACHES 64
struct KeepCaches {
    char* at[KEEP_CACHES];
};
struct KeepArgs {
    DraftRows dr;
    const int* block_table;      // [R, max_blocks]
    const int* parents;          // [T]
    const int* tokens;           // [T]
    const int* chosen;           // [T]
    int* counts;                 // [R], null: written by another launch
    int* path;                   // [R, max_rows]
    int* fresh;                  // [R, max_rows]
    int* err;
    int max_blocks, pages, outer, page_size, inner;     // a cache is [pages, outer, page, inner pieces]
    int n_caches;
};

template <typename V>
__global__ void __launch_bounds__(KEEP_THREADS) keep_drafts_kernel(const KeepArgs a, const __grid_constant__ KeepCaches caches) {
    extern __shared__ int shared[];
    __shared__ int s_count, s_first;
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x, tid = threadIdx.x, most = a.dr.max_rows;
    int* next = shared;                                               // [n]: the child that is confirmed
    int* path = shared + most;                                        // [n]
    int row0, start;
    const int n = draft_rows(a.dr, r, row0, start);
    for (int i = tid; i < n; i += KEEP_THREADS) next[i] = 0x7fffffff;
    __syncthreads();
    for (int i = tid; i < n; i += KEEP_THREADS) {
        const int parent = a.parents[row0 + i];
        if (i > 0 && parent >= 0 && parent < i && a.tokens[row0 + i] == a.chosen[row0 + parent]) atomicMin(next + parent, i);
    }
    __syncthreads();
    if (tid == 0) {
        int count = 0, first = n, node = 0;
        if (n > 0)
            for (;;) {
                if (node != count && first == n) first = count;       // moves from here on
                path[count++] = node;
                node = next[node];
                if (node == 0x7fffffff) break;
            }
        s_count = count;
        s_first = min(first, count);
    }
    __syncthreads();
    const int count = s_count, first = s_first, moves = count - first;
    if (blockIdx.y == 0 && a.counts) {
        if (tid == 0) a.counts[r] = count;
        for (int k = tid; k < most; k += KEEP_THREADS) {
            a.path[(size_t)r * most + k] = k < count ? path[k] : -1;
            a.fresh[(size_t)r * most + k] = k < count ? a.chosen[row0 + path[k]] : -1;
        }
    }
    if (moves == 0) return;
    // the rows that move, of a cache's outer index 0: from, to; -1: a place that the cache does not have
    const size_t page_rows = (size_t)a.outer * a.page_size;
    auto row_of = [&](long long e) -> long long {
        if (e >= (long long)a.max_blocks * a.page_size) { atomicCAS(a.err, 0, RG_BAD_PAGE); return -1; }
        const int page = a.block_table[(size_t)r * a.max_blocks + e / a.page_size];
        if ((unsigned)page >= (unsigned)a.pages) { atomicCAS(a.err, 0, RG_BAD_PAGE); return -1; }
        return (long long)page * (long long)page_rows + e % a.page_size;
    };
    __shared__ long long from[KEEP_AHEAD], to[KEEP_AHEAD];
    const long long columns = (long long)a.n_caches * a.outer * a.inner;
    for (int k0 = first; k0 < count; k0 += KEEP_AHEAD) {
        __syncthreads();
        if (tid < KEEP_AHEAD) {
            const int k = k0 + tid;
            const bool there = k < count;
            const long long f = there ? row_of((long long)start + path[k]) : -1, t = there ? row_of((long long)start + k) : -1;
            from[tid] = t < 0 ? -1 : f;
            to[tid] = t;
        }
        __syncthreads();
        for (long long col = (long long)blockIdx.y * KEEP_THREADS + tid; col < columns; col += (long long)gridDim.y * KEEP_THREADS) {
            const int c = (int)(col % a.inner), lo = (int)(col / a.inner), cache = lo / a.outer, o = lo % a.outer;
            V* base = reinterpret_cast<V*>(caches.at[cache]) + (size_t)o * a.page_size * a.inner + c;
            V v[KEEP_AHEAD];
#pragma unroll
            for (int j = 0; j < KEEP_AHEAD; ++j)
                if (from[j] >= 0) v[j] = base[from[j] * a.inner];
#pragma unroll
            for (int j = 0; j < KEEP_AHEAD; ++j)
                if (from[j] >= 0) base[to[j] * a.inner] = v[j];
        }
    }
}

// `piece`: bytes (1, 2, 4, 8 or 16) that rows and addresses are multiples of; inner: pieces of a row.
extern "C" int rg_keep_drafts(const unsigned long long* caches, int n_caches, int pages, int outer, int page_size, int inner, int piece,
                              const int* block_table, int max_blocks, const int* cu_rows, const int* starts, const int* parents, const int* tokens,
                              const int* chosen, int R, int T, int max_rows, int* counts, int* path, int* fresh, int sms, int* err, void* stream) {
    if (R <= 0) return 0;
    if (n_caches < 1 || pages < 0 || outer < 1 || page_size < 1 || inner < 1 || max_blocks < 0 || max_rows < 0 || max_rows > DRAFT_MOST || sms < 1)
        return RG_ERR_UNSUPPORTED;
    const size_t smem = 2 * (size_t)max_rows * sizeof(int);
    for (int c0 = 0; c0 < n_caches; c0 += KEEP_CACHES) {
        KeepCaches at = {};
        const int some = n_caches - c0 < KEEP_CACHES ? n_caches - c0 : KEEP_CACHES;
        for (int i = 0; i < some; ++i) {
            if (caches[c0 + i] % piece) return RG_ERR_UNSUPPORTED;
            at.at[i] = reinterpret_cast<char*>(caches[c0 + i]);
        }
        const KeepArgs a = {{cu_rows, starts, R, T, max_rows}, block_table, parents, tokens, chosen, c0 ? nullptr : counts, path, fresh, err,
                            max_blocks, pages, outer, page_size, inner, some};
        const long long columns = (long long)some * outer * inner, needed = (columns + KEEP_THREADS - 1) / KEEP_THREADS;
        const long long room = (8ll * sms + R - 1) / R;
        const dim3 grid((unsigned)R, (unsigned)(needed < room ? needed : (room > 0 ? room : 1)));
        int e;
        switch (piece) {
            case 16: e = rg_launch(keep_drafts_kernel<uint4>, grid, dim3(KEEP_THREADS), smem, (cudaStream_t)stream, 1, a, at); break;
            case 8: e = rg_launch(keep_drafts_kernel<uint2>, grid, dim3(KEEP_THREADS), smem, (cudaStream_t)stream, 1, a, at); break;
            case 4: e = rg_launch(keep_drafts_kernel<unsigned>, grid, dim3(KEEP_THREADS), smem, (cudaStream_t)stream, 1, a, at); break;
            case 2: e = rg_launch(keep_drafts_kernel<unsigned short>, grid, dim3(KEEP_THREADS), smem, (cudaStream_t)stream, 1, a, at); break;
            case 1: e = rg_launch(keep_drafts_kernel<unsigned char>, grid, dim3(KEEP_THREADS), smem, (cudaStream_t)stream, 1, a, at); break;
            default: return RG_ERR_UNSUPPORTED;
        }
        if (e) return e;
    }
    return 0;
}
