// What the kernels of attention_parts.cu and attention_prefix_tcgen05.cu share: how a launch's blocks are cut out of rows
// and entries, and where a part of a softmax is left.
//
// Rows (single tokens) attend two lists of cached entries: the prefix of their group, which the group's rows share, and
// entries of their own; either may be empty.  Both are read through block tables, entry e at row e % page_size of page
// table[e / page_size].  A list is cut into parts of `per` entries; a part leaves, per row and head, the unnormalised
// output o = sum_e 2^(s_e - m) v_e with its m = max_e s_e and l = sum_e 2^(s_e - m), s = scale log2(e) q.k, in 32-bit:
//   out = sum_parts 2^(m - M) o / sum_parts 2^(m - M) l,   M = max_parts m
// A prefix is read once for up to as many queries (rows x heads of one kv head) as a block takes, instead of once a row.
#pragma once
#include "common.cuh"

struct PartArgs {
    const void* q;               // [T, q_stride]: head h of row t at q[t * q_stride + h * d]
    const void* kv;              // [pages, 2, nkv, page_size, d]
    const int* block_table;      // [T, max_blocks]: a row's own entries
    const int* positions;        // [T]: row t sees its own entries 0 .. positions[t] (-1: none)
    const int* prefix_table;     // [n_groups, prefix_blocks]
    const int* groups;           // [n_groups][3]: first row, rows, entries of the prefix; in order of rows
    float* part_o;               // [T, nh, slots, d]
    float* part_ml;              // [T, nh, slots, 2]
    float* scores;               // null, or [T, nh, score_ld]: s of every own entry
    long long score_ld;
    int q_stride, max_blocks, prefix_blocks, n_groups;
    int prefix_parts, prefix_per, own_parts, own_per;   // parts of either list and entries a part
    int prefix_tiles, own_tiles;                        // query tiles of a group, of a row's kv head
    int prefix_limit, own_limit;                        // the most entries that the call says, and that tables, parts and scratch have room for
    int max_rows;                                       // rows of a group that a launch is sized for
    int T, nh, nkv, d, page_size, page_shift;           // page_shift: log2 of the page size, or -1
    float scale_log2;
    int beside;                  // the kernel before this one writes nothing that this one reads, and the other way round
};

// One block's share: the queries [q0, q0 + nq) of (first row, kv head), query i being row row0 + i / group, head
// kvh * group + i % group; the entries [e0, e1) of `table`; the slot where the part is left.
struct PartShare {
    const int* table;
    int row0, kvh, q0, nq, e0, e1, slot;
};

// How many entries of its own row t sees, and how many group g's prefix has; never more than there is room for.
__device__ __forceinline__ int own_entries(const PartArgs& a, int t) { return min(a.positions[t] + 1, a.own_limit); }
__device__ __forceinline__ int prefix_entries(const PartArgs& a, int g) { return min(a.groups[g * 3 + 2], a.prefix_limit); }
// Rows of group g: no more than a launch is sized for.
__device__ __forceinline__ int group_rows(const PartArgs& a, int g) {
    const int row0 = a.groups[g * 3];
    return row0 < 0 ? 0 : min(min(a.groups[g * 3 + 1], a.max_rows), a.T - row0);
}

// Block b of a launch: the prefixes' parts first, their blocks numbered part by part within (tile, kv head, group).
// false: there is nothing to do (a shorter prefix or fewer rows than the launch was sized for).
__device__ __forceinline__ bool part_share(const PartArgs& a, int tile_queries, int b, PartShare& s) {
    const int group = a.nh / a.nkv;
    const int prefix_blocks = a.n_groups * a.nkv * a.prefix_tiles * a.prefix_parts;
    if (b < prefix_blocks) {
        const int part = b % a.prefix_parts, tile = b / a.prefix_parts % a.prefix_tiles;
        const int gk = b / a.prefix_parts / a.prefix_tiles, g = gk / a.nkv;
        s.row0 = a.groups[g * 3];
        const int rows = group_rows(a, g), entries = prefix_entries(a, g);
        s.kvh = gk % a.nkv;
        s.q0 = tile * tile_queries;
        s.nq = min(tile_queries, rows * group - s.q0);
        s.e0 = part * a.prefix_per;
        s.e1 = min(entries, s.e0 + a.prefix_per);
        s.slot = part;
        s.table = a.prefix_table + (size_t)g * a.prefix_blocks;
    } else {
        b -= prefix_blocks;
        const int part = b % a.own_parts, tile = b / a.own_parts % a.own_tiles, tk = b / a.own_parts / a.own_tiles;
        s.row0 = tk / a.nkv;
        s.kvh = tk % a.nkv;
        s.q0 = tile * tile_queries;
        s.nq = min(tile_queries, group - s.q0);
        s.e0 = part * a.own_per;
        s.e1 = min(own_entries(a, s.row0), s.e0 + a.own_per);
        s.slot = a.prefix_parts + part;
        s.table = a.block_table + (size_t)s.row0 * a.max_blocks;
    }
    return s.nq > 0 && s.e0 < s.e1;
}
__host__ __device__ inline long long part_blocks(const PartArgs& a) {
    return ((long long)a.n_groups * a.nkv * a.prefix_tiles * a.prefix_parts) + (long long)a.T * a.nkv * a.own_tiles * a.own_parts;
}

// How many parts row t has of either list.
__device__ __forceinline__ int own_parts_at(const PartArgs& a, int position) {
    return (max(0, min(position + 1, a.own_limit)) + a.own_per - 1) / a.own_per;
}
__device__ __forceinline__ int own_parts_of(const PartArgs& a, int t) { return own_parts_at(a, a.positions[t]); }
// Row t's group (-1: none), and how many entries its prefix has.  Whole warps, all lanes for the same row: a lane looks at every 32nd
// group, the first group that has the row counts; a group's three numbers are asked for together.  (One group after the other in every
// thread: 48 groups of 4 rows on 64 shared and 32 own entries, 32 heads on 8 of 128, 35.1 us, 22.9 so; 1,000 of 2 rows, 8 heads on 2
// of 64, 384 and 45.9; one group 8.7 and 8.6.)
__device__ __forceinline__ int group_of(const PartArgs& a, int t, int& entries) {
    const int lane = threadIdx.x & 31;
    int g0 = 0, e = 0;
    unsigned hit = 0;
#pragma unroll 1
    for (; !hit && g0 < a.n_groups; g0 += 32) {
        const int g = g0 + lane;
        const int* at = a.groups + 3 * (size_t)min(g, a.n_groups - 1);
        const int row0 = at[0], rows = at[1];
        e = at[2];
        const int i = t - row0;
        hit = __ballot_sync(0xffffffffu, g < a.n_groups && row0 >= 0 && i >= 0 && i < min(rows, a.max_rows));
    }
    const int first = __ffs(hit) - 1;
    entries = hit ? max(0, min(__shfl_sync(0xffffffffu, e, first), a.prefix_limit)) : 0;
    return hit ? g0 - 32 + first : -1;
}
// Its table, where there are entries.
__device__ __forceinline__ const int* prefix_of(const PartArgs& a, int t, int& entries) {
    const int g = group_of(a, t, entries);
    return a.prefix_table + (size_t)max(g, 0) * a.prefix_blocks;
}
__device__ __forceinline__ int prefix_parts_of(const PartArgs& a, int t) {
    int entries;
    group_of(a, t, entries);
    return (entries + a.prefix_per - 1) / a.prefix_per;
}
