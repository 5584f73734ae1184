// Eviction from the paged cache by accumulated attention weight.
//
// Request r holds n = lens[r] entries; of each kv head's, k = min(n, keep[r]) stay: the greatest by weight, ties to the lowest
// entry, where an entry whose place in the text is below protect_first or above positions[r] - protect_last (or whose weight is
// no number) counts as +infinity.  The entries that stay need no order (attention has none), so only those behind the new
// length move: the i-th of them goes into the i-th entry before it that got free.  Sources lie at k and beyond, destinations
// before k: the moves of K and V rows are independent of one another, and of the fewest bytes there can be.
//
// One cluster per (request, kv head).  The k-th greatest key is found by three passes over its bits (11, 11 and 10, from
// the top): a histogram in shared memory, added up over the cluster, and a sum from the top bin down.  Then every warp walks
// consecutive entries, 32 at a time, and numbers ties, free entries and late ones by ballots, with the counts of the warps and
// blocks before it.  Lists of destinations and sources go through global scratch (they stay in L2); the cluster's warps then
// move a row each.
#include "common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

#define EV_THREADS 512
#define EV_WARPS (EV_THREADS / 32)
#define EV_BINS 2048

struct EvictArgs {
    void* kv;                    // [pages, 2, nkv, page_size, d], `row_bytes` a row
    const float* weights;        // [n_slots, nkv, ld]
    const int* places;           // [n_slots, nkv, ld]
    float* weights_out;
    int* places_out;
    const int* slots;            // [R]
    const int* block_table;      // [R, max_blocks]
    const int* lens;             // [R]
    const int* keep;             // [R]
    const int* positions;        // [R]: the place of the newest token
    int* new_lens;               // [R]
    int* moves;                  // [R * nkv][2][limit / 2 + 1]: destinations, sources
    long long ld;
    int n_slots, max_blocks, R, nkv, page_size, row_bytes, protect_first, protect_last, limit;
};

// A weight as an unsigned number of the same order.
__device__ __forceinline__ uint32_t weight_key(const EvictArgs& a, float w, int place, int newest) {
    if (place < a.protect_first || place > newest - a.protect_last || w != w) w = INFINITY;
    const uint32_t b = __float_as_uint(w + 0.f);                    // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sum over the block's threads, by thread; total: of all.  scratch: EV_WARPS + 1 ints.
__device__ __forceinline__ int block_scan(int v, int* scratch, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < EV_WARPS; ++w) {
        const int c = scratch[w];
        if (w < warp) before += c;
        total += c;
    }
    return before + s - v;
}

template <bool CACHED>          // the block's keys fit its shared memory
__global__ void __launch_bounds__(EV_THREADS) evict_kernel(const EvictArgs a) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[EV_BINS], scan[EV_WARPS + 1], found[3], counts[4];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    // No early start for the kernel behind this one: attention kernels ask for cached keys ahead of their own wait.
    pdl_wait();
    const int row = blockIdx.x / C, r = row / a.nkv, h = row % a.nkv;
    const int slot = a.slots[r], n = min(a.lens[r], a.limit), k = min(n, max(0, a.keep[r])), newest = a.positions[r];
    if (slot < 0 || slot >= a.n_slots || n <= 0) {                  // the same for the whole cluster
        if (h == 0 && rank == 0 && threadIdx.x == 0) a.new_lens[r] = a.lens[r];
        return;
    }
    if (h == 0 && rank == 0 && threadIdx.x == 0) a.new_lens[r] = k;
    const size_t base = ((size_t)slot * a.nkv + h) * a.ld;
    const float* w = a.weights + base;
    const int* places = a.places + base;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // this block's entries, in runs of whole warps: [c0, c1), a warp's share `run` of them
    const int run = ((n + C * EV_WARPS - 1) / (C * EV_WARPS) + 31) & ~31;
    const int c0 = min(n, rank * run * EV_WARPS), c1 = min(n, c0 + run * EV_WARPS);
    auto key_of = [&](int e) -> uint32_t { return CACHED ? keys[e - c0] : weight_key(a, w[e], places[e], newest); };
    int *dst = a.moves + (size_t)row * 2 * (a.limit / 2 + 1), *src = dst + a.limit / 2 + 1;
    int n_moves = 0;
    if (k < n) {
        if (CACHED) {
            for (int e = c0 + tid; e < c1; e += EV_THREADS) keys[e - c0] = weight_key(a, w[e], places[e], newest);
        }
        // the k-th greatest key: `high` its bits so far, `left` how many of the entries with these bits stay
        uint32_t high = 0;
        int left = k;
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
            __syncthreads();
            for (int e = c0 + tid; e < c1; e += EV_THREADS) {
                const uint32_t key = key_of(e);
                if (pass == 0 || key >> (shift + bits) == high >> (shift + bits)) atomicAdd(&hist[key >> shift & ((1 << bits) - 1)], 1);
            }
            cluster.sync();
            // bins from the top down, 4 a thread; only counts that are whole numbers are added: any order gives the same
            int c[EV_BINS / EV_THREADS], mine = 0, total;
#pragma unroll
            for (int j = 0; j < EV_BINS / EV_THREADS; ++j) {
                const int bin = EV_BINS - 1 - (tid * (EV_BINS / EV_THREADS) + j);
                c[j] = 0;
                for (int q = 0; q < C; ++q) c[j] += cluster.map_shared_rank(hist, q)[bin];
                mine += c[j];
            }
            int above = block_scan(mine, scan, total);
#pragma unroll
            for (int j = 0; j < EV_BINS / EV_THREADS; ++j) {
                if (above < left && left <= above + c[j]) {
                    found[0] = EV_BINS - 1 - (tid * (EV_BINS / EV_THREADS) + j);
                    found[1] = left - above;
                }
                above += c[j];
            }
            cluster.sync();                                         // histograms are read, `found` is there
            if (k > 0) { high |= (uint32_t)found[0] << shift; left = found[1]; }
        }
        // k = 0: nothing stays, and no bin is found
        const uint32_t kth = k > 0 ? high : 0xffffffffu;
        // Ties before each entry: counts of the blocks and warps before, then ballots.
        const int w0 = min(c1, c0 + warp * run), w1 = min(c1, w0 + run);
        auto before_me = [&](int mine, int which) -> int {          // the sum of `mine` (a warp's) over all warps before this one
            int total;
            const int in_block = block_scan(lane == 0 ? mine : 0, scan, total);
            if (tid == 0) counts[which] = total;
            cluster.sync();
            int sum = __shfl_sync(0xffffffffu, in_block, 0);
            for (int q = 0; q < rank; ++q) sum += cluster.map_shared_rank(counts, q)[which];
            return sum;
        };
        int ties = 0;
        for (int e = w0 + lane; e - lane < w1; e += 32) ties += __popc(__ballot_sync(0xffffffffu, e < w1 && key_of(e) == kth));
        int tie = before_me(ties, 0);
        // which entries stay; how many of this warp's get free or come late
        int free_n = 0, late_n = 0, t2 = tie;
        auto stays = [&](int e, int& t) -> bool {
            const uint32_t key = e < w1 ? key_of(e) : 0u;
            const bool eq = e < w1 && key == kth;
            const uint32_t all = __ballot_sync(0xffffffffu, eq);
            const bool in = e < w1 && (key > kth || (eq && t + __popc(all & ((1u << lane) - 1)) < left)) && k > 0;
            t += __popc(all);
            return in;
        };
        for (int e = w0 + lane; e - lane < w1; e += 32) {
            const bool in = stays(e, t2);
            free_n += __popc(__ballot_sync(0xffffffffu, e < w1 && e < k && !in));
            late_n += __popc(__ballot_sync(0xffffffffu, e < w1 && e >= k && in));
        }
        int free_at = before_me(free_n, 1), late_at = before_me(late_n, 2);
        for (int e = w0 + lane; e - lane < w1; e += 32) {
            const bool in = stays(e, tie), gone = e < w1 && e < k && !in, late = e < w1 && e >= k && in;
            const uint32_t f = __ballot_sync(0xffffffffu, gone), l = __ballot_sync(0xffffffffu, late);
            if (gone) dst[free_at + __popc(f & ((1u << lane) - 1))] = e;
            if (late) src[late_at + __popc(l & ((1u << lane) - 1))] = e;
            free_at += __popc(f);
            late_at += __popc(l);
            if (in && e < k) {
                a.weights_out[base + e] = w[e];
                a.places_out[base + e] = places[e];
            }
        }
        __threadfence();
        cluster.sync();                                             // the lists are whole
        for (int q = 0; q < C; ++q) n_moves += cluster.map_shared_rank(counts, q)[2];
        cluster.sync();                                             // nobody leaves while its counts are read
    } else {
        for (int e = c0 + tid; e < c1; e += EV_THREADS) {
            a.weights_out[base + e] = w[e];
            a.places_out[base + e] = places[e];
        }
    }
    // The moves, a warp each.
    const int* table = a.block_table + (size_t)r * a.max_blocks;
    const size_t half = (size_t)a.nkv * a.page_size * a.row_bytes;  // bytes of a page's keys, or values
    auto at = [&](int e) -> unsigned char* {
        return (unsigned char*)a.kv + (size_t)table[e / a.page_size] * 2 * half + ((size_t)h * a.page_size + e % a.page_size) * a.row_bytes;
    };
    for (int i = rank * EV_WARPS + warp; i < n_moves; i += C * EV_WARPS) {
        const int to = __ldcg(dst + i), from = __ldcg(src + i);
        unsigned char *pt = at(to), *pf = at(from);
        if (a.row_bytes % 16 == 0 && ((uintptr_t)a.kv & 15) == 0) {
            const int n16 = a.row_bytes / 16;
            for (int j = lane; j < 2 * n16; j += 32) {
                const size_t off = j < n16 ? (size_t)j * 16 : half + (size_t)(j - n16) * 16;
                *reinterpret_cast<uint4*>(pt + off) = *reinterpret_cast<const uint4*>(pf + off);
            }
        } else {
            for (int j = lane; j < a.row_bytes; j += 32) {           // rows of 2 or 4 bytes an element
                pt[j] = pf[j];
                pt[half + j] = pf[half + j];
            }
        }
        if (lane == 0) {
            a.weights_out[base + to] = w[from];
            a.places_out[base + to] = places[from];
        }
    }
    __threadfence();
}

#define EV_MOST_KEYS 48000      // that fit a block's shared memory beside the rest

// moves: scratch of R * nkv * 2 * (max_context / 2 + 1) ints.  cluster: blocks a (request, kv head), 1, 2, 4 or 8.
extern "C" int rg_evict_entries(void* kv, int elem_bytes, const float* weights, const int* places, float* weights_out, int* places_out,
                                int ld, int n_slots, const int* slots, const int* block_table, int max_blocks, const int* lens,
                                const int* keep, const int* positions, int* new_lens, int R, int nkv, int d, int page_size,
                                int protect_first, int protect_last, int max_context, int* moves, int cluster, void* stream) {
    if (R <= 0) return 0;
    if (nkv < 1 || d < 1 || page_size < 1 || max_context < 1 || max_context > ld || cluster < 1 || cluster > 8 || (cluster & (cluster - 1)) ||
        (long long)R * nkv * cluster > 0x7fffffffll)
        return RG_ERR_UNSUPPORTED;
    const int limit = max_context;
    const EvictArgs a = {kv, weights, places, weights_out, places_out, slots, block_table, lens, keep, positions, new_lens, moves, ld, n_slots,
                         max_blocks, R, nkv, page_size, d * elem_bytes, protect_first, protect_last,
                         (int)min((long long)limit, (long long)max_blocks * page_size)};
    const long long a_warp = ((((long long)limit + cluster * EV_WARPS - 1) / (cluster * EV_WARPS)) + 31) / 32 * 32;
    const long long most = a_warp * EV_WARPS;
    const bool cached = most <= EV_MOST_KEYS;
    const size_t smem = cached ? (size_t)most * 4 : 0;
    void (*kernel)(EvictArgs) = cached ? evict_kernel<true> : evict_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return rg_launch(kernel, dim3((unsigned)(R * nkv * cluster)), dim3(EV_THREADS), smem, (cudaStream_t)stream, cluster, a);
}
