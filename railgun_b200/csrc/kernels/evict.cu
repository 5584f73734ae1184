// Eviction from the paged cache by accumulated attention weight.
//
// Request r holds n = lens[r] entries; of each kv head's, k = min(n, keep[r]) stay: the greatest by weight, ties to the lowest
// entry, where an entry whose place in the text is below protect_first or above positions[r] - protect_last (or whose weight is
// no number) counts as +infinity.  The entries that stay need no order (attention has none), so only those behind the new
// length move: the i-th of them goes into the i-th entry before it that got free.  Sources lie at k and beyond, destinations
// before k: the moves of K and V rows are independent of one another, and of the fewest bytes there can be.
//
// One block per (request, kv head), or a cluster of them.  A warp holds consecutive entries' keys, a key of each run of 32 a
// lane, in registers.  The k-th greatest key is found digit by digit from the top (10 bits a digit, or 12 where a block holds
// many keys): a histogram of the keys that agree so far, in shared memory, added up over the cluster, and a sum from the top
// bin down; once at most 128 keys agree they are compared with one another.  (Cutting the interval in four with three counts
// a step needs 7 to 8 steps to get there: 14 us of 53 for clusters of two on 16,384 keys.)  Then free entries and late ones
// are numbered by ballots, with the counts of the warps and blocks before.  A warp takes up to 32 moves at a time: their
// addresses a lane each, then their rows in 16-byte pieces, several a lane under way.
//
// What bounds it: the digits, one after the other, each a barrier or three away from the next; then, with many moves, memory.  8 prompts
// of 8,192 to 16,384 entries down to 2,048 in 8 kv heads of 128: 40 us, 15 of them the choice, 24 the moves of 83 MB (3.4 TB/s
// from a cold cache); 64 requests of 1,040 down to 1,024 in 8 heads of 64: 9.7 us, one launch.
#include "common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

struct EvictArgs {
    void* kv;                    // [pages, 2, nkv, page_size, d], `row_bytes` a row
    const float* weights;        // [n_slots, nkv, ld]
    const int* places;           // [n_slots, nkv, ld]
    float* weights_out;          // may be the weights themselves, and so the places
    int* places_out;
    const int* slots;            // [R]
    const int* block_table;      // [R, max_blocks]
    const int* lens;             // [R]
    const int* keep;             // [R]
    const int* positions;        // [R]: the place of the newest token
    int* new_lens;               // [R]
    int* moves;                  // [R * nkv][ev_list(limit)]: how many, destinations, sources
    long long ld;
    int n_slots, max_blocks, R, nkv, page_size, row_bytes, protect_first, protect_last, limit;
};

__host__ __device__ inline size_t ev_list(int limit) { return 1 + 2 * ((size_t)limit / 2 + 1); }

// A weight as an unsigned number of the same order.
__device__ __forceinline__ uint32_t weight_key(const EvictArgs& a, float w, int place, int newest) {
    if (place < a.protect_first || place > newest - a.protect_last || w != w) w = INFINITY;
    const uint32_t b = __float_as_uint(w + 0.f);                    // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sums over warps: what every warp's lane 0 gives, for all warps of the block (cluster).
template <int WARPS, int N, bool CLUSTERED>
struct Sums {
    int (*all)[WARPS][N];        // shared memory, two of them in turn: one barrier a sum
    int turn;
    // total: over all; before: over the warps before this one, of blocks before this one as well
    __device__ __forceinline__ void of(const int (&mine)[N], int (&total)[N], int (&before)[N]) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        int (*now)[N] = all[turn];
        turn ^= 1;
        if (lane < N) {
            int v = mine[0];
#pragma unroll
            for (int i = 1; i < N; ++i) v = lane == i ? mine[i] : v;
            now[warp][lane] = v;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) total[i] = before[i] = 0;
        auto add = [&](const int (*from)[N], bool earlier) {         // a warp's numbers a lane, then over the lanes
            const int w = lane < WARPS ? lane : 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int v = lane < WARPS ? from[w][i] : 0;
                total[i] += __reduce_add_sync(0xffffffffu, v);
                before[i] += __reduce_add_sync(0xffffffffu, earlier || (from == now && lane < warp) ? v : 0);
            }
        };
        if constexpr (CLUSTERED) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            for (int q = 0; q < (int)cluster.num_blocks(); ++q) {
                if (q == (int)cluster.block_rank()) add(now, false);
                else add(cluster.map_shared_rank(now, q), q < (int)cluster.block_rank());
            }
        } else {
            __syncthreads();
            add(now, false);
        }
    }
};

// Moves of row (request, kv head) `row` by the warp `mover` of `movers`: `batch` (up to 32) at a time, a lane each for their addresses.  Rows are
// pieces of 16 bytes, K and V one after the other; or, where they are not made of those, bytes.
template <int DEEP>                  // pieces a lane under way
__device__ __forceinline__ void move_rows(const EvictArgs& a, int row, const int* dst, const int* src, int n_moves, int mover, int movers, int batch) {
    const int lane = threadIdx.x & 31, r = row / a.nkv, h = row % a.nkv;
    const size_t base = ((size_t)a.slots[r] * a.nkv + h) * a.ld;
    const int* table = a.block_table + (size_t)r * a.max_blocks;
    const size_t half = (size_t)a.nkv * a.page_size * a.row_bytes;   // bytes of a page's keys, or values
    const bool wide = a.row_bytes % 16 == 0 && ((uintptr_t)a.kv & 15) == 0;
    auto at = [&](int e) -> size_t {
        return (size_t)__ldg(table + e / a.page_size) * 2 * half + ((size_t)h * a.page_size + e % a.page_size) * a.row_bytes;
    };
    unsigned char* kv = (unsigned char*)a.kv;
    // `lanes` of the warp share a move, `side` moves side by side: a power of two that fits its pieces
    int lanes = 32;
    while (lanes > 1 && (wide ? a.row_bytes / 8 : 2 * a.row_bytes) % lanes) lanes >>= 1;
    const int side = 32 / lanes;
    for (int i0 = mover * batch; i0 < n_moves; i0 += movers * batch) {
        const int m = min(batch, n_moves - i0);
        long long to = 0, from = 0;
        if (lane < m) {
            const int e = dst[i0 + lane], f = src[i0 + lane];
            to = (long long)at(e);
            from = (long long)at(f);
            a.weights_out[base + e] = __ldcg(a.weights + base + f);
            a.places_out[base + e] = __ldcg(a.places + base + f);
        }
        const int row_pieces = wide ? a.row_bytes / 16 : a.row_bytes;
        for (int c = lane & (lanes - 1); c < 2 * row_pieces; c += lanes) {
            unsigned char* mine = kv + (c < row_pieces ? (size_t)c : half / (wide ? 16 : 1) + (c - row_pieces)) * (wide ? 16 : 1);
            for (int k0 = 0; k0 < m; k0 += DEEP * side) {
                uint4 v[DEEP];
#pragma unroll
                for (int j = 0; j < DEEP; ++j) {
                    const int k = k0 + j * side + lane / lanes;
                    const unsigned char* get = mine + __shfl_sync(0xffffffffu, from, k < m ? k : 0);
                    if (k < m) {
                        if (wide) v[j] = *reinterpret_cast<const uint4*>(get);
                        else v[j].x = *get;
                    }
                }
#pragma unroll
                for (int j = 0; j < DEEP; ++j) {
                    const int k = k0 + j * side + lane / lanes;
                    unsigned char* put = mine + __shfl_sync(0xffffffffu, to, k < m ? k : 0);
                    if (k < m) {
                        if (wide) *reinterpret_cast<uint4*>(put) = v[j];
                        else *put = (unsigned char)v[j].x;
                    }
                }
            }
        }
    }
}

#define EV_FEW 128                // keys that are compared with one another
// bits of a digit: four bins a thread
__host__ __device__ constexpr int ev_bits(int threads) { return threads == 256 ? 10 : 12; }

// PER: keys a thread holds; 0: they are made anew whenever one is asked for.  FUSED: the block makes the moves, too.
template <int THREADS, int PER, bool CLUSTERED, bool FUSED>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 4 : 1) evict_kernel(const EvictArgs a) {
    constexpr int WARPS = THREADS / 32, BITS = ev_bits(THREADS), BINS = 1 << BITS;
    static_assert(BINS == 4 * THREADS, "four bins a thread");
    static_assert(!(CLUSTERED && FUSED), "a cluster's lists are in global memory");
    extern __shared__ __align__(16) int lists[];                     // destinations and sources, where the block itself moves
    __shared__ __align__(16) int hist[2][BINS];                      // of two digits in turn
    __shared__ int sums_of[2][WARPS][2], scan[WARPS], found[3], few_n, kth_is[3];
    __shared__ uint32_t few[EV_FEW];
    const int C = CLUSTERED ? (int)cg::this_cluster().num_blocks() : 1, rank = CLUSTERED ? (int)cg::this_cluster().block_rank() : 0;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    reinterpret_cast<int4*>(hist[0])[tid] = make_int4(0, 0, 0, 0);
    reinterpret_cast<int4*>(hist[1])[tid] = make_int4(0, 0, 0, 0);
    if (tid == 0) few_n = 0;
    // No early start for the kernel behind this one: attention kernels ask for cached keys ahead of their own wait.
    pdl_wait();
    const int row = blockIdx.x / C, r = row / a.nkv, h = row % a.nkv;
    const int slot = a.slots[r], n = a.lens[r], k = min(n, max(0, a.keep[r])), newest = a.positions[r];
    // Left alone, the same for the whole cluster; also a request with more entries than there is room for: its newest ones would go
    // without having been looked at.
    const bool alone = slot < 0 || slot >= a.n_slots || n <= 0 || n > a.limit;
    if (h == 0 && rank == 0 && tid == 0) a.new_lens[r] = alone ? n : k;
    if (alone) {                                                      // the kernel that moves goes by the number of moves
        if constexpr (!FUSED)
            if (rank == 0 && tid == 0) a.moves[(size_t)row * ev_list(a.limit)] = 0;
        return;
    }
    const size_t base = ((size_t)slot * a.nkv + h) * a.ld;
    const float* w = a.weights + base;
    const int* places = a.places + base;
    // this warp's entries: `run` runs of 32 from w0 on
    const int run = (n + C * THREADS - 1) / (C * THREADS), w0 = (rank * WARPS + warp) * run * 32;
    uint32_t held[PER ? PER : 1];
    if constexpr (PER > 0) {
#pragma unroll
        for (int j0 = 0; j0 < PER; j0 += 8) {                        // eight of each under way: as many as there are registers for
            float wv[8];
            int pv[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = min(w0 + (j0 + j) * 32 + lane, n - 1);   // no branch: the loads leave together
                wv[j] = __ldcg(w + e);
                pv[j] = __ldcg(places + e);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) held[j0 + j] = weight_key(a, wv[j], pv[j], newest);
        }
    }
    // What lies before the new length, as if it stayed (moves come over it); in place it is there already, and what moves
    // comes from where nothing is written.
    if (a.weights_out != a.weights || a.places_out != a.places)
        for (int e = rank * THREADS + tid; e < k; e += C * THREADS) {
            a.weights_out[base + e] = __ldcg(w + e);
            a.places_out[base + e] = __ldcg(places + e);
        }
    // f(entry, its key, is there such an entry): for every run of the warp, all lanes together
    auto each = [&](auto f) {
        if constexpr (PER > 0) {
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (j < run) { const int e = w0 + j * 32 + lane; f(e, held[j], e < n); }
        } else {
            for (int j = 0; j < run; ++j) {
                const int e = w0 + j * 32 + lane;
                f(e, e < n ? weight_key(a, __ldcg(w + e), __ldcg(places + e), newest) : 0u, e < n);
            }
        }
    };
    auto block_or_cluster_sync = [&]() {
        if constexpr (CLUSTERED) cg::this_cluster().sync();
        else __syncthreads();
    };
    Sums<WARPS, 2, CLUSTERED> sums = {sums_of, 0};
    int n_moves = 0;
    int *dst = FUSED ? lists : a.moves + (size_t)row * ev_list(a.limit) + 1, *src = dst + a.limit / 2 + 1;
    if (k < n) {
        // The k-th greatest key has the digits of `high` down to bit `shift`; of the `in` keys that have them `left` stay.
        uint32_t high = 0;
        int shift = 32, left = k, in = n;
        block_or_cluster_sync();
        for (int digit = 0; shift > 0 && in > EV_FEW && k > 0; ++digit) {
            const int bits = min(BITS, shift), was = shift;
            shift -= bits;
            int* mine = hist[digit & 1];
            each([&](int, uint32_t key, bool there) {
                if (there && (was == 32 || key >> was == high >> was)) atomicAdd(&mine[key >> shift & ((1 << bits) - 1)], 1);
            });
            block_or_cluster_sync();
            // bins from the top down, four a thread; counts are whole numbers: any order of adding gives the same
            const int at = THREADS - 1 - tid;
            int4 c = make_int4(0, 0, 0, 0);
            for (int q = 0; q < C; ++q) {
                const int4* from = reinterpret_cast<const int4*>(mine);
                if constexpr (CLUSTERED) from = cg::this_cluster().map_shared_rank(from, q);
                const int4 x = from[at];
                c.x += x.x; c.y += x.y; c.z += x.z; c.w += x.w;
            }
            const int sum = c.x + c.y + c.z + c.w;
            int s = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += u;
            }
            if (lane == 31) scan[warp] = s;
            __syncthreads();
            const int earlier = __reduce_add_sync(0xffffffffu, lane < warp && lane < WARPS ? scan[lane] : 0);
            int above = earlier + s - sum;
            if (above < left && left <= above + sum) {                 // one thread's bins hold it
                int bin = 4 * at + 3, here = c.w;
                if (left > above + here) { above += here; --bin; here = c.z; }
                if (left > above + here) { above += here; --bin; here = c.y; }
                if (left > above + here) { above += here; --bin; here = c.x; }
                found[0] = bin;
                found[1] = left - above;
                found[2] = here;
            }
            block_or_cluster_sync();                                   // histograms are read, `found` is there
            high |= (uint32_t)found[0] << shift;
            left = found[1];
            in = found[2];
            if (digit + 2 < (32 + BITS - 1) / BITS) reinterpret_cast<int4*>(mine)[tid] = make_int4(0, 0, 0, 0);   // for the digit after the next
        }
        int equal = in;                                                // keys that are the one itself, once all digits are there
        if (shift > 0 && k > 0) {
            // few enough: a key with g greater ones and q equal ones is the one if g < left <= g + q
            each([&](int, uint32_t key, bool there) {
                if (there && (shift == 32 || key >> shift == high >> shift)) {
                    if constexpr (CLUSTERED) {
                        cg::cluster_group cluster = cg::this_cluster();
                        cluster.map_shared_rank(few, 0)[atomicAdd(cluster.map_shared_rank(&few_n, 0), 1)] = key;
                    } else few[atomicAdd(&few_n, 1)] = key;
                }
            });
            if constexpr (CLUSTERED) {
                cg::this_cluster().sync();
                if (rank > 0 && tid < in) few[tid] = cg::this_cluster().map_shared_rank(few, 0)[tid];
            }
            __syncthreads();
            // a candidate a warp at a time, compared with all of them by the lanes
            for (int i = warp; i < in; i += WARPS) {
                const uint32_t mine = few[i];
                int c = 0;                                             // greater, and equal << 16
#pragma unroll
                for (int j = 0; j < EV_FEW / 32; ++j) {
                    const uint32_t other = few[lane + 32 * j];
                    if (lane + 32 * j < in) c += (other > mine ? 1 : 0) + (other == mine ? 1 << 16 : 0);
                }
                c = __reduce_add_sync(0xffffffffu, c);
                const int g = c & 0xffff, q = c >> 16;
                if (lane == 0 && g < left && left <= g + q) { kth_is[0] = (int)mine; kth_is[1] = left - g; kth_is[2] = q; }
            }
            __syncthreads();
            high = (uint32_t)kth_is[0];
            left = kth_is[1];
            equal = kth_is[2];
        }
        // What stays: keys above `high`, and of those that equal it the first `left`.  Bit j: the entry of run j stays.
        const bool some = k > 0 && left < equal;                       // only some of the equal ones: they are numbered
        int total[2], before[2], c[2] = {0, 0}, tie = 0;
        if (some) {
            each([&](int, uint32_t key, bool there) { c[0] += __popc(__ballot_sync(0xffffffffu, there && key == high)); });
            sums.of(c, total, before);
            tie = before[0];
        }
        const uint32_t below = (1u << lane) - 1;
        auto stays = [&](uint32_t key, bool there, int& t) -> bool {
            if (!some) return there && key >= high && k > 0;
            const uint32_t all = __ballot_sync(0xffffffffu, there && key == high);
            const bool in = there && (key > high || (key == high && t + __popc(all & below) < left));
            t += __popc(all);
            return in;
        };
        int t2 = tie;
        c[0] = c[1] = 0;                                               // free, late: this lane's, then the warp's
        each([&](int e, uint32_t key, bool there) {
            const bool in = stays(key, there, t2);
            c[0] += there && e < k && !in;
            c[1] += e >= k && in;
        });
#pragma unroll
        for (int i = 0; i < 2; ++i) c[i] = __reduce_add_sync(0xffffffffu, c[i]);
        sums.of(c, total, before);
        n_moves = total[1];
        each([&](int e, uint32_t key, bool there) {
            const bool in = stays(key, there, tie), front = e < k, moves = there && in != front;
            const uint32_t m = __ballot_sync(0xffffffffu, moves), f = __ballot_sync(0xffffffffu, front) & m, l = m & ~f;
            if (moves) (front ? dst : src)[front ? before[0] + __popc(f & below) : before[1] + __popc(l & below)] = e;
            before[0] += __popc(f);
            before[1] += __popc(l);
        });
        block_or_cluster_sync();                                       // the lists are whole, and nobody reads another block's sums any more
    }
    if constexpr (FUSED) move_rows<4>(a, row, dst, src, n_moves, warp, WARPS, min(32, (n_moves + WARPS - 1) / WARPS));
    else if (rank == 0 && tid == 0) a.moves[(size_t)row * ev_list(a.limit)] = n_moves;
    if constexpr (FUSED) __threadfence();
}

// The moves of a row that evict_kernel has listed.  (Bulk copies through shared memory, a row each, are slower, 48 us for the
// whole of eight prompts against 39: the unit that makes them is bound by their number.)  grid (blocks that share a row's moves, R * nkv)
#define EV_MOVERS 2               // blocks an SM
__global__ void __launch_bounds__(256, EV_MOVERS) evict_moves_kernel(const EvictArgs a) {
    pdl_wait();                                                      // no early start for the kernel behind, as above
    const int* list = a.moves + (size_t)blockIdx.y * ev_list(a.limit);
    const int n = list[0], movers = gridDim.x * 8;
    move_rows<8>(a, blockIdx.y, list + 1, list + 2 + a.limit / 2, n, blockIdx.x * 8 + (threadIdx.x >> 5), movers,
                 min(32, (n + movers - 1) / movers));
    __threadfence();
}

// moves: scratch of R * nkv * (2 * (max_context / 2) + 3) ints where max_context is above 2,048.  cluster: blocks a (request, kv
// head), 1, 2, 4 or 8; one holds up to 16,384 keys.
extern "C" int rg_evict_entries(void* kv, int elem_bytes, const float* weights, const int* places, float* weights_out, int* places_out,
                                int ld, int n_slots, const int* slots, const int* block_table, int max_blocks, const int* lens,
                                const int* keep, const int* positions, int* new_lens, int R, int nkv, int d, int page_size,
                                int protect_first, int protect_last, int max_context, int* moves, int cluster, int sms, void* stream) {
    if (R <= 0) return 0;
    if (nkv < 1 || d < 1 || page_size < 1 || max_context < 1 || max_context > ld || cluster < 1 || cluster > 8 || (cluster & (cluster - 1)) ||
        (long long)R * nkv * cluster > 0x7fffffffll || (max_context > 256 * 8 && (long long)R * nkv > 65535))
        return RG_ERR_UNSUPPORTED;
    const int limit = (int)min((long long)max_context, (long long)max_blocks * page_size);
    const EvictArgs a = {kv, weights, places, weights_out, places_out, slots, block_table, lens, keep, positions, new_lens, moves, ld, n_slots,
                         max_blocks, R, nkv, page_size, d * elem_bytes, protect_first, protect_last, limit};
    // Up to 2,048 entries 256 threads hold the keys and make the moves.  Above, a thousand threads hold up to 16,384, a cluster up to
    // eight times as many, and the moves are a second kernel's, so that all SMs take part however few heads there are (64 heads of
    // 8,192 to 16,384 entries, 2,048 of which stay: 39 us, 44 with clusters of two that move what they have chosen).
    const unsigned rows = (unsigned)(R * nkv);
#define RG_EV(T, P, CL, FU, SMEM) e = rg_launch(evict_kernel<T, P, CL, FU>, dim3(rows * (CL ? cluster : 1)), dim3(T), SMEM, s, CL ? cluster : 1, a)
    const cudaStream_t s = (cudaStream_t)stream;
    int e;
    if (max_context <= 256 * 8) {
        RG_EV(256, 8, false, true, 2 * (limit / 2 + 1) * sizeof(int));
        return e;
    }
    if (cluster == 1) {
        if (limit > 1024 * 16) return RG_ERR_UNSUPPORTED;
        RG_EV(1024, 16, false, false, 0);
    } else if (limit <= cluster * 1024 * 16) RG_EV(1024, 16, true, false, 0);
    else RG_EV(1024, 0, true, false, 0);
#undef RG_EV
    if (e) return e;
    const int share = max(1, min((limit / 2 + 31) / 32, sms * EV_MOVERS / (int)rows));
    return rg_launch(evict_moves_kernel, dim3(share, rows), dim3(256), 0, s, 1, a);
}
