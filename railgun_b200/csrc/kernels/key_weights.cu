// The weights that cached entries receive from portions of prompts:
//   w[e] (+)= sum over the portion's rows t at positions p_t >= e and the heads h of a kv head of 2^(s_th(e) - z_th),
//   s = scale log2(e) q.k,   z_th = log2 sum_e 2^(s_th(e))
// in two passes over the scores: z first, then the sums.  A block of the second pass owns its entries and goes over all
// rows that see them, so sums have one order and need no atomics.
#include "packed_f32.cuh"
#include "tcgen05.cuh"
#include <type_traits>

struct WeightArgs {
    const void* q;               // [T, q_stride]: head h of row t at q[t * q_stride + h * d]
    const void* kv;              // [pages, 2, nkv, page_size, d]
    const int* block_table;      // [R, max_blocks]
    const int* cu_rows;          // [R + 1]: request r's rows are cu_rows[r] .. cu_rows[r + 1] - 1
    const int* starts;           // [R]: the position of its first row; row i sees entries 0 .. starts[r] + i
    const int* fresh;            // [R]: entries from here on have no earlier weight
    const int* slots;            // [R]: where its weights are (negative: nowhere)
    float* weights;              // [n_slots, nkv, weights_ld]
    float* z;                    // [T, nh]
    long long weights_ld;
    int q_stride, max_blocks, n_slots, T, R, nh, nkv, d, page_size, limit;   // limit: the most entries there is room for
    float scale_log2;
    int max_rows;                // the most rows of a request
};

// Request r's rows and entries, cut to what there is room for.
__device__ __forceinline__ void rows_of(const WeightArgs& a, int r, int& row0, int& rows, int& start, int& entries) {
    row0 = max(0, a.cu_rows[r]);
    rows = min(min(a.cu_rows[r + 1], a.T) - row0, a.max_rows);
    start = a.starts[r];
    entries = rows > 0 && start >= 0 ? min(start + rows, a.limit) : 0;
}

// A pass of which parts are joined afterwards.
struct KtArgs {
    WeightArgs w;
    float* part_ml;              // [T, nh, row_parts, 2]
    float* part_w;               // [parts of the second pass, R, nkv, limit]; null: the weights themselves are written
    int row_parts, parts;        // of the first pass, and of this one: what streams, dealt out in turn
    // the tensor cores' kernel
    int* err;
    int blocks, n_items;         // 256 lanes each, of the longest request
    int tile_rows;               // rows of a query tile: 128 / group
    int page_shift;
};

// ---------------------------------------------------------------------------------------------------
// Any head size up to 256, any page size, 32-bit or bfloat16 storage, all arithmetic in 32-bit.  16 or 64 queries (rows x heads
// of a kv head) by 64 entries at a time, 2 x 4 or 8 x 4 a thread: eight of them read 12 quads of shared memory for 128
// multiply-adds, two of them 6 for 32.  What bounds it is arithmetic, and with few blocks the trip to memory before every tile:
// 32-bit, 32 heads on 8 of 128, 256 rows 58 us, 2,048 rows 1.6 ms (21 TFLOP/s over both passes).  (16 queries at a time, single
// numbers loaded and one block for all rows that see a tile: 691 us for the 256 rows.)
// ---------------------------------------------------------------------------------------------------
#define KW_THREADS 128
#define KW_K 64
#define KW_FEW 32                  // queries a kv head up to which 16 at a time waste less than they read

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load4(const bf16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}

// ROWS rows of d numbers, from `at` (-1: zeros), times f; to rows of ld, zeros up to the next four columns.
template <typename A, bool VEC, int ROWS>
__device__ __forceinline__ void load_rows(float* to, int ld, int d, const A* from, const long long* at, float f) {
    const int pieces = VEC ? d / 4 : (d + 3) & ~3, step = KW_THREADS / pieces, odd = KW_THREADS - step * pieces;
#pragma unroll 4
    for (int row = threadIdx.x / pieces, p = threadIdx.x % pieces; row < ROWS; p += odd, row += step) {
        if (p >= pieces) { p -= pieces; if (++row >= ROWS) break; }
        const long long x = at[row];
        if (VEC) {
            float4 v = {0.f, 0.f, 0.f, 0.f};
            if (x >= 0) v = load4(from + x + 4 * p);
            *reinterpret_cast<float4*>(to + row * ld + 4 * p) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
        } else to[row * ld + p] = x >= 0 && p < d ? to_f32(from[x + p]) * f : 0.f;
    }
}
// Where query qi of (request's first row, kv head) and entry e are.
__device__ __forceinline__ long long query_at(const WeightArgs& a, int row0, int kvh, int qi) {
    const int group = a.nh / a.nkv;
    return (long long)(row0 + qi / group) * a.q_stride + (kvh * group + qi % group) * a.d;
}
__device__ __forceinline__ long long key_at(const WeightArgs& a, const int* table, int kvh, int e) {
    return (long long)table[e / a.page_size] * 2 * a.nkv * a.page_size * a.d + ((long long)kvh * a.page_size + e % a.page_size) * a.d;
}
template <int QI>
__device__ __forceinline__ void tile_scores(float (&sc)[QI][4], const float* qs, const float* ks, int ld, int d, int qa, int ka) {
#pragma unroll
    for (int i = 0; i < QI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
#pragma unroll 2
    for (int c = 0; c < d; c += 4) {
        float4 k4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const float4*>(ks + (ka + 16 * j) * ld + c);
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const float4 q4 = *reinterpret_cast<const float4*>(qs + (QI * qa + i) * ld + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sc[i][j] += q4.x * k4[j].x; sc[i][j] += q4.y * k4[j].y;
                sc[i][j] += q4.z * k4[j].z; sc[i][j] += q4.w * k4[j].w;
            }
        }
    }
}

__host__ __device__ inline int kw_row(int d) { return ((d + 3) & ~3) + 4; }
static size_t kw_smem(int d, int queries) { return (size_t)((queries + KW_K) * kw_row(d) + 8 * KW_K) * sizeof(float); }

// grid (query tiles x parts of the entries, nkv, R)
template <typename A, bool VEC, int QI>
__global__ void __launch_bounds__(KW_THREADS) row_sums_general_kernel(const KtArgs k) {
    extern __shared__ __align__(16) float smem[];
    constexpr int QT = 8 * QI;
    __shared__ long long at[KW_K];
    static_assert(QT <= KW_K, "the queries' places fit");
    const WeightArgs& a = k.w;
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y, group = a.nh / a.nkv, q0 = blockIdx.x / k.parts * QT, part = blockIdx.x % k.parts, tid = threadIdx.x;
    int row0, rows, start, entries;
    rows_of(a, r, row0, rows, start, entries);
    const int nq = min(QT, rows * group - q0);
    if (nq <= 0 || entries <= 0) return;
    const int ld = kw_row(a.d), qa = tid >> 4, ka = tid & 15;
    float *qs = smem, *ks = smem + QT * ld;
    if (tid < QT) at[tid] = tid < nq ? query_at(a, row0, kvh, q0 + tid) : -1;
    __syncthreads();
    load_rows<A, VEC, QT>(qs, ld, a.d, (const A*)a.q, at, a.scale_log2);
    const int* table = a.block_table + (size_t)r * a.max_blocks;
    const int last = min(entries, start + (q0 + nq - 1) / group + 1);          // what the tile's last row sees
    auto look_up = [&](int e0) -> long long { return tid < KW_K && e0 + tid < last ? key_at(a, table, kvh, e0 + tid) : -1; };
    long long at_next = look_up(part * KW_K);
    float m[QI], l[QI];
#pragma unroll
    for (int i = 0; i < QI; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
    for (int e0 = part * KW_K; e0 < last; e0 += k.parts * KW_K) {
        __syncthreads();                                             // the last tile is read
        if (tid < KW_K) at[tid] = at_next;
        __syncthreads();
        load_rows<A, VEC, KW_K>(ks, ld, a.d, (const A*)a.kv, at, 1.f);
        at_next = look_up(e0 + k.parts * KW_K);
        __syncthreads();
        float sc[QI][4];
        tile_scores<QI>(sc, qs, ks, ld, a.d, qa, ka);
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int sees = min(last, start + (q0 + QI * qa + i) / group + 1) - e0;
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (ka + 16 * j >= sees) sc[i][j] = -INFINITY;
                mx = fmaxf(mx, sc[i][j]);
            }
            const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn;
            float sum = l[i] * exp2f(m[i] - ms);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += exp2f(sc[i][j] - ms);
            l[i] = sum;
            m[i] = mn;
        }
    }
#pragma unroll
    for (int i = 0; i < QI; ++i) {
        float M = m[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float ms = M == -INFINITY ? 0.f : M;
        float L = l[i] * exp2f(m[i] - ms);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        const int qi = q0 + QI * qa + i;
        if (ka == 0 && QI * qa + i < nq) {
            const size_t to = (size_t)(row0 + qi / group) * a.nh + kvh * group + qi % group;
            if (k.parts > 1) *reinterpret_cast<float2*>(k.part_ml + (to * k.parts + part) * 2) = make_float2(M, L);
            else a.z[to] = L == 0.f ? INFINITY : ms + log2f(L);       // no weight at all: every 2^(s - z) is 0
        }
    }
}

// grid (tiles of entries x parts of the queries, nkv, R)
template <typename A, bool VEC, int QI>
__global__ void __launch_bounds__(KW_THREADS) entry_sums_general_kernel(const KtArgs k) {
    extern __shared__ __align__(16) float smem[];
    constexpr int QT = 8 * QI;
    __shared__ long long at[KW_K];
    const WeightArgs& a = k.w;
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y, group = a.nh / a.nkv, e0 = blockIdx.x / k.parts * KW_K, part = blockIdx.x % k.parts, tid = threadIdx.x;
    const int slot = a.slots[r];
    int row0, rows, start, entries;
    rows_of(a, r, row0, rows, start, entries);
    const int n = min(KW_K, entries - e0);
    if (n <= 0 || slot < 0 || slot >= a.n_slots) return;
    const int ld = kw_row(a.d), qa = tid >> 4, ka = tid & 15;
    float *qs = smem, *ks = qs + QT * ld, *sums = ks + KW_K * ld;              // sums [8][64]
    if (tid < KW_K) at[tid] = tid < n ? key_at(a, a.block_table + (size_t)r * a.max_blocks, kvh, e0 + tid) : -1;
    __syncthreads();
    load_rows<A, VEC, KW_K>(ks, ld, a.d, (const A*)a.kv, at, 1.f);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int q0 = max(0, e0 - start) * group + part * QT; q0 < rows * group; q0 += k.parts * QT) {  // from the first row that sees entry e0
        __syncthreads();
        if (tid < QT) at[tid] = q0 + tid < rows * group ? query_at(a, row0, kvh, q0 + tid) : -1;
        __syncthreads();
        load_rows<A, VEC, QT>(qs, ld, a.d, (const A*)a.q, at, a.scale_log2);
        float z[QI];
        int sees[QI];
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            const int qi = q0 + QI * qa + i;
            const bool query = qi < rows * group;
            z[i] = query ? a.z[(size_t)(row0 + qi / group) * a.nh + kvh * group + qi % group] : 0.f;
            sees[i] = query ? start + qi / group + 1 - e0 : 0;
        }
        __syncthreads();
        float sc[QI][4];
        tile_scores<QI>(sc, qs, ks, ld, a.d, qa, ka);
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (ka + 16 * j < sees[i]) sum[j] += exp2f(sc[i][j] - z[i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[qa * KW_K + ka + 16 * j] = sum[j];
    __syncthreads();
    if (tid < n) {
        float added = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) added += sums[i * KW_K + tid];
        const int e = e0 + tid;
        if (k.part_w) k.part_w[(((size_t)part * a.R + r) * a.nkv + kvh) * a.limit + e] = added;
        else {
            float* w = a.weights + ((size_t)slot * a.nkv + kvh) * a.weights_ld + e;
            *w = (e < a.fresh[r] ? *w : 0.f) + added;
        }
    }
}

// ---------------------------------------------------------------------------------------------------
// bfloat16, head sizes 64 and 128, up to 128 heads a kv head, pages of 8 tokens or a larger power of two: the 5th-generation
// tensor cores.  Both passes have one structure and differ in what stays and what streams:
//   row sums:    128 lanes = queries (rows x heads of a kv head), keys stream by;   m, l of a row run in its thread
//   entry sums:  128 lanes = entries, queries stream by;   w[e] is a sum over columns, again inside a thread: no exchange
// A block has two such tiles of 128 (a "side" each: its own accumulator, issuing warp and four warps of exponentials), which
// share the streamed tiles, so a streamed tile is fetched once for 256 lanes; where only one tile is left, the sides take
// every other streamed tile of it.  Per streamed tile of 128 and side: S = A B^T in 128 columns of tensor memory, two
// buffers a side, then one pass of exponentials over it while the tensor core works on the next.  Blocks are persistent:
// items (kv head, 256 lanes, part of what streams) are dealt out to and fro, the heaviest first.  Two loading warps work out
// what an item is, look up its pages and fetch its first tiles while earlier ones are worked on (a ring of items); loads,
// products and exponentials run on across items.  (One warp that looked up one item and one tile at a time: the last 1 to 33 rows
// of 8 prompts 57 us, 54 now; 8,192 rows 861, 779 now.)
//
// What bounds it: one 2^x an element and pass.  128 x 128 of them take 1,024 cycles of a scheduler's MUFU, the products of a
// tile 520 of the tensor core (head size 128).  The MUFU is busy for six tenths of a pass, waits for a tile's scores and uneven items
// take the rest: 2,048 rows of 32 heads on 8 of 128 70 us, 8,192 rows 779 (353 TFLOP/s counted once, twice that are done).  The
// last 1 to 33 rows of 8 prompts of 3,000 to 6,000 entries at head size 64 54 us: a lane without a query still costs a 2^x.
// (Entries as lanes and queries as columns in both passes, with sums over columns in registers: 110.)
// ---------------------------------------------------------------------------------------------------
#define KT_THREADS 384             // warps 0-3, 4-7: sides 0, 1; 8, 11: TMA; 9, 10: MMA issue of sides 0, 1 (9: tensor memory)
#define KT_TILE 128
__host__ __device__ constexpr int kt_a_stages(int pieces) { return pieces == 1 ? 4 : 2; }      // of two tiles each
__host__ __device__ constexpr int kt_b_stages(int pieces) { return pieces == 1 ? 4 : 2; }

struct alignas(16) KtItem {             // read in quads
    int r, kvh, part, row0, rows, start, entries;
    int m0, n_m;                 // first lane tile, how many of the two there are (0: the end)
    int b0, n_b;                 // streamed tiles b0, b0 + parts, ..
    int slot, fresh;
};

template <bool ENTRIES>
__device__ __forceinline__ bool kt_item(const KtArgs& a, int i, KtItem& t) {
    const int per_block = a.w.R * a.w.nkv * a.parts, blk = i / per_block, rest = i % per_block;
    t.part = rest % a.parts;
    t.kvh = rest / a.parts % a.w.nkv;
    t.r = rest / a.parts / a.w.nkv;
    rows_of(a.w, t.r, t.row0, t.rows, t.start, t.entries);
    t.slot = ENTRIES ? a.w.slots[t.r] : 0;
    t.fresh = ENTRIES ? a.w.fresh[t.r] : 0;
    if (t.entries <= 0) return false;
    const int q_tiles = (t.rows + a.tile_rows - 1) / a.tile_rows;
    if (ENTRIES) {
        t.m0 = 2 * blk;                                             // the first entries are seen by the most rows
        t.n_m = min(2, (t.entries + KT_TILE - 1) / KT_TILE - t.m0);
        t.b0 = max(0, t.m0 * KT_TILE - t.start) / a.tile_rows;
        t.n_b = q_tiles - t.b0;
    } else {
        t.m0 = 2 * (a.blocks - 1 - blk);                            // the last rows see the most entries
        t.n_m = min(2, q_tiles - t.m0);
        const int last_row = min(t.rows, (t.m0 + 2) * a.tile_rows) - 1;
        t.b0 = 0;
        t.n_b = (min(t.entries, t.start + last_row + 1) + KT_TILE - 1) / KT_TILE;
    }
    t.n_b = t.n_b > t.part ? (t.n_b - t.part + a.parts - 1) / a.parts : 0;
    t.b0 += t.part;
    return t.n_m > 0 && (!ENTRIES || a.part_w || (t.slot >= 0 && t.slot < a.w.n_slots));
}

// q_map: 64 columns x heads x rows, a box of 64 x group x tile_rows; kv_map: the cache as rows of the head size, a box of
// min(page, 128) rows x 64 columns.
template <int PIECES, bool ENTRIES>
__global__ void __launch_bounds__(KT_THREADS, 1)
key_weights_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const KtArgs a) {
    extern __shared__ unsigned char smem_raw[];
    constexpr int NA = kt_a_stages(PIECES), NB = kt_b_stages(PIECES);
    constexpr uint32_t PIECE = KT_TILE * 128, TILE = PIECE * PIECES;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u, sA = base, sB = sA + 2 * NA * TILE;   // NA stages of two tiles; NB tiles
    __shared__ __align__(8) uint64_t bars[3 * NA + 2 * NB + 8 + 2];
    // -z of a streamed tile's columns and their positions: a copy for every warp, so that warps wait for nothing but tiles
    __shared__ __align__(16) float col_z[ENTRIES ? 8 : 1][2][KT_TILE];
    __shared__ __align__(16) int col_p[ENTRIES ? 8 : 1][2][KT_TILE];
    __shared__ float other_ml[ENTRIES ? 1 : KT_TILE][2];             // side 1's results for side 0, where they share a tile
    __shared__ KtItem items[NA];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    // i_full: an item; a_full: its lane tiles as well; s_full, s_empty: side 0's two buffers, side 1's; x_full, x_empty: other_ml
    const uint32_t i_full = smem_addr(bars), a_full = i_full + 8 * NA, a_empty = a_full + 8 * NA, b_full = a_empty + 8 * NA, b_empty = b_full + 8 * NB,
                   s_full = b_empty + 8 * NB, s_empty = s_full + 32, x_full = s_empty + 32, x_empty = x_full + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.w.nh / a.w.nkv;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < NA; ++i) { mbar_init(i_full + 8 * i, 1); mbar_init(a_full + 8 * i, 1); mbar_init(a_empty + 8 * i, 2 + 8); }   // both issuers, eight warps
        for (int i = 0; i < NB; ++i) { mbar_init(b_full + 8 * i, 1); mbar_init(b_empty + 8 * i, 2); }
        for (int i = 0; i < 4; ++i) { mbar_init(s_full + 8 * i, 1); mbar_init(s_empty + 8 * i, KT_TILE); }
        mbar_init(x_full, KT_TILE);
        mbar_init(x_empty, KT_TILE);
        fence_barrier_init();
    }
    if (warp == 9) tmem_alloc(&tmem_slot, 512u);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;                                 // side g, buffer b: columns 256 g + 128 b
    pdl_wait();
    pdl_trigger();
    bool ok = true;
    KtItem t = {};
    // Does side g work on streamed tile b of this item?  With one lane tile the sides take turns.
    auto mine_is = [&](int g, int b) -> bool { return t.n_m == 2 || (ENTRIES ? g == 0 : (b & 1) == g); };
    if (warp == 8 || warp == 11) {
        // ---- loads.  Both warps walk through the items, each issues half of the boxes (one takes some 85 cycles of a warp).
        const int half = warp == 11;
        const int box_rows = min(a.w.page_size, KT_TILE), boxes = KT_TILE / box_rows, box = lane % boxes, piece = lane / boxes;
        const bool mine = piece < PIECES && (ENTRIES || (lane & 1) == half);   // a box of a piece of the head each
        // Items are looked up by all lanes, 32 of this block's rounds at a time, and page ids asked for an item, or four streamed
        // tiles, ahead: a look-up takes as long as a tile's exponentials.
        KtItem held = {}, n = {};
        int r0 = -32;
        uint32_t left = 0;
        auto next_item = [&]() {
            while (left == 0) {
                r0 += 32;
                if ((long long)r0 * gridDim.x >= a.n_items) { n = KtItem{}; return; }
                // to and fro: who got the heaviest of one round gets the lightest of the next
                const int i = (r0 + lane) * gridDim.x + (lane & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                left = __ballot_sync(0xffffffffu, i < a.n_items && kt_item<ENTRIES>(a, i, held));
            }
            const int from = __ffs(left) - 1;
            left &= left - 1;
            auto get = [&](int v) -> int { return __shfl_sync(0xffffffffu, v, from); };
            n.r = get(held.r); n.kvh = get(held.kvh); n.part = get(held.part); n.row0 = get(held.row0); n.rows = get(held.rows);
            n.start = get(held.start); n.entries = get(held.entries); n.m0 = get(held.m0); n.n_m = get(held.n_m); n.b0 = get(held.b0);
            n.n_b = get(held.n_b); n.slot = get(held.slot); n.fresh = get(held.fresh);
        };
        auto page_of = [&](const KtItem& x, int tile) -> int {       // behind the entries: any page
            const int e = tile * KT_TILE + box * box_rows;
            return x.n_b > 0 ? a.w.block_table[(size_t)x.r * a.w.max_blocks + (e < x.entries ? e >> a.page_shift : 0)] : 0;
        };
        constexpr int AHEAD = ENTRIES ? 1 : 4;
        auto first_pages = [&](const KtItem& x, int (&page)[AHEAD]) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) page[j] = page_of(x, ENTRIES ? x.m0 + (x.n_m == 2 ? half : 0) : x.b0 + j * a.parts);
        };
        auto load_keys = [&](uint32_t dst, uint32_t bar, int tile, int page) {
            const int e = tile * KT_TILE + box * box_rows;
            if (mine)
                tma_load_2d(dst + piece * PIECE + box * box_rows * 128, &kv_map, bar, 64 * piece,
                            (page * 2 * a.w.nkv + t.kvh) * a.w.page_size + (e & (a.w.page_size - 1)));
        };
        auto load_queries = [&](uint32_t dst, uint32_t bar, int tile) {
            if (lane < PIECES) tma_load_3d(dst + lane * PIECE, &q_map, bar, 64 * lane, t.kvh * group, t.row0 + tile * a.tile_rows);
        };
        const uint32_t q_bytes = (uint32_t)(PIECES * 128 * group * a.tile_rows);
        const uint32_t a_bytes = ENTRIES ? TILE : q_bytes, b_bytes = ENTRIES ? q_bytes : TILE;
        int page[AHEAD], bi = 0;
        next_item();
        first_pages(n, page);
        for (int ai = 0; ok; ++ai) {
            t = n;
            const int sa = ai % NA;
            if (ai >= NA) ok = mbar_wait_all(a_empty + 8 * sa, ((ai / NA) & 1) ^ 1, a.err, 71, &abort_flag);
            if (!ok) break;
            if (half == 0 && lane == 0) {
                items[sa] = t;
                mbar_arrive(i_full + 8 * sa);
                if (t.n_b) mbar_expect_tx(a_full + 8 * sa, (uint32_t)t.n_m * a_bytes);
                else mbar_arrive(a_full + 8 * sa);
            }
            __syncwarp();
            if (t.n_m == 0) break;                                   // the end
            if (t.n_b && half < t.n_m) {                             // a lane tile each
                if (ENTRIES) load_keys(sA + (2 * sa + half) * TILE, a_full + 8 * sa, t.m0 + half, page[0]);
                else load_queries(sA + (2 * sa + half) * TILE, a_full + 8 * sa, t.m0 + half);
            }
            next_item();
            if (ENTRIES || t.n_b == 0) first_pages(n, page);
            for (int b0 = 0; b0 < t.n_b && ok; b0 += AHEAD) {
                int page_next[AHEAD];
                if (!ENTRIES) {
                    if (b0 + AHEAD >= t.n_b) first_pages(n, page_next);
                    else
#pragma unroll
                        for (int j = 0; j < AHEAD; ++j) page_next[j] = page_of(t, t.b0 + (b0 + AHEAD + j) * a.parts);
                }
#pragma unroll
                for (int j = 0; j < AHEAD; ++j) {
                    if (b0 + j >= t.n_b || !ok) break;
                    const int sb = bi % NB, tile = t.b0 + (b0 + j) * a.parts;
                    if (!ENTRIES || half == 0) {
                        if (bi >= NB) ok = mbar_wait_all(b_empty + 8 * sb, ((bi / NB) & 1) ^ 1, a.err, 72, &abort_flag);
                        if (!ok) break;
                        if (half == 0 && lane == 0) mbar_expect_tx(b_full + 8 * sb, b_bytes);
                        __syncwarp();
                        if (ENTRIES) load_queries(sB + sb * TILE, b_full + 8 * sb, tile);
                        else load_keys(sB + sb * TILE, b_full + 8 * sb, tile, page[j]);
                    }
                    ++bi;
                }
#pragma unroll
                for (int j = 0; j < AHEAD; ++j)
                    if (!ENTRIES) page[j] = page_next[j];
            }
        }
    } else if (warp == 9 || warp == 10) {
        // ---- products of a side: the whole warp walks and waits, one elected lane issues
        constexpr uint32_t idesc = make_idesc(KT_TILE, KT_TILE, false);
        const int g = warp - 9;
        const bool issuer = elect_one();
        int si = 0, bi = 0;                                          // tiles of this side; streamed tiles
        for (int ai = 0; ok; ++ai) {
            const int sa = ai % NA;
            ok = mbar_wait_all(a_full + 8 * sa, (ai / NA) & 1, a.err, 73, &abort_flag);
            if (!ok) break;
            t.n_m = items[sa].n_m;
            t.n_b = items[sa].n_b;
            if (t.n_m == 0) break;
            const uint32_t at = sA + (2 * sa + (t.n_m == 2 ? g : 0)) * TILE;
            for (int b = 0; b < t.n_b && ok; ++b, ++bi) {
                const int sb = bi % NB;
                ok = mbar_wait_all(b_full + 8 * sb, (bi / NB) & 1, a.err, 74, &abort_flag);
                if (ok && mine_is(g, b)) {
                    const int buf = si & 1;
                    if (si > 1) ok = mbar_wait_all(s_empty + 16 * g + 8 * buf, ((si >> 1) & 1) ^ 1, a.err, 75, &abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    if (issuer) {
#pragma unroll
                        for (int x = 0; x < PIECES; ++x) {
                            const uint64_t ad = desc_k_major(at + x * PIECE), bd = desc_k_major(sB + sb * TILE + x * PIECE);
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                tc_mma(tmem + 256u * g + 128u * buf, ad + 2u * k, bd + 2u * k, idesc, x + k > 0 ? 1u : 0u);
                        }
                        tc_commit(s_full + 16 * g + 8 * buf);
                        tc_commit(b_empty + 8 * sb);
                    }
                    ++si;
                } else if (ok && lane == 0) mbar_arrive(b_empty + 8 * sb);
                __syncwarp();
            }
            if (!ok) break;
            if (issuer) tc_commit(a_empty + 8 * sa);                 // once every product of the item is done
            __syncwarp();
        }
    } else if (warp < 8) {
        // ---- exponentials: thread = lane of the accumulator
        const int g = warp >> 2, row = threadIdx.x & 127;
        const uint32_t tmem_row = tmem + 256u * g + ((uint32_t)((warp & 3) * 32) << 16);
        const uint64_t scale2 = pack2(a.w.scale_log2, a.w.scale_log2);
        int si = 0, ai = 0, xi = 0;
        auto next_item = [&](KtItem& to) -> bool {
            if (!mbar_wait_all(i_full + 8 * (ai % NA), (ai / NA) & 1, a.err, 78, &abort_flag)) return false;
            to = items[ai % NA];
            __syncwarp();
            if (lane == 0) mbar_arrive(a_empty + 8 * (ai % NA));
            ++ai;
            return true;
        };
        if (ENTRIES) {
            // columns lane + 32 j of a streamed tile: their queries' z and positions (-1: no query)
            float z_next[4];
            int p_next[4];
            KtItem n = {};
            float before_next = 0.f;
            int c_row[4], c_z[4];                                    // their rows in the tile, and where z is from the tile's first row's on
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = lane + 32 * j;
                c_row[j] = c < a.tile_rows * group ? c / group : 0x3fffffff;
                c_z[j] = c / group * a.w.nh + c % group;
            }
            auto columns = [&](const KtItem& x, int b) {
                const int r0 = (x.b0 + b * a.parts) * a.tile_rows, rows = g < x.n_m && b < x.n_b ? x.rows - r0 : 0;
                const float* z = a.w.z + (size_t)(x.row0 + r0) * a.w.nh + x.kvh * group;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    p_next[j] = c_row[j] < rows ? x.start + r0 + c_row[j] : -1;
                    z_next[j] = c_row[j] < rows ? z[c_z[j]] : 0.f;
                }
            };
            auto place = [&](const KtItem& x) -> float* { return a.w.weights + ((size_t)x.slot * a.w.nkv + x.kvh) * a.w.weights_ld; };
            // the next item, and what of it takes a trip to memory: asked for while this one's last tile is worked on
            auto look_ahead = [&]() -> bool {
                if (!next_item(n)) return false;
                columns(n, 0);
                const int e = (n.m0 + g) * KT_TILE + row;
                before_next = !a.part_w && g < n.n_m && e < min(n.entries, n.fresh) ? place(n)[e] : 0.f;
                return true;
            };
            ok = look_ahead();
            while (ok && n.n_m > 0) {
                t = n;
                const float before = before_next;
                const bool there = g < t.n_m;
                const int e = (t.m0 + g) * KT_TILE + row;
                uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
                if (t.n_b == 0 || !there) ok = look_ahead();
                for (int b = 0; b < t.n_b && there && ok; ++b, ++si) {
                    const int buf = si & 1;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        col_z[warp][buf][lane + 32 * j] = -z_next[j];
                        col_p[warp][buf][lane + 32 * j] = p_next[j];
                    }
                    __syncwarp();                                    // they are there (and every lane is done with those before)
                    if (b + 1 < t.n_b) columns(t, b + 1);
                    else ok = look_ahead();
                    if (ok) ok = mbar_wait_all(s_full + 16 * g + 8 * buf, (si >> 1) & 1, a.err, 76, &abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    const float4* z4 = reinterpret_cast<const float4*>(col_z[warp][buf]);
                    const int4* p4 = reinterpret_cast<const int4*>(col_p[warp][buf]);
                    const int r0 = (t.b0 + b * a.parts) * a.tile_rows, cols = min(a.tile_rows, t.rows - r0) * group;
                    // every column a query that sees every entry of this tile?
                    const bool edge = cols < KT_TILE || t.start + r0 < (t.m0 + g + 1) * KT_TILE - 1;
                    uint32_t v[2][32];
                    auto chunk = [&](auto edge_c, int c, const uint32_t (&x)[32]) {
                        constexpr bool EDGE = decltype(edge_c)::value;
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 z = z4[(32 * c + j) >> 2];
                            float y[4];
                            unpack2(fma2(pack2(__uint_as_float(x[j]), __uint_as_float(x[j + 1])), scale2, pack2(z.x, z.y)), y[0], y[1]);
                            unpack2(fma2(pack2(__uint_as_float(x[j + 2]), __uint_as_float(x[j + 3])), scale2, pack2(z.z, z.w)), y[2], y[3]);
                            if (EDGE) {
                                const int4 p = p4[(32 * c + j) >> 2];
                                if (p.x < e) y[0] = -INFINITY;
                                if (p.y < e) y[1] = -INFINITY;
                                if (p.z < e) y[2] = -INFINITY;
                                if (p.w < e) y[3] = -INFINITY;
                            }
                            sum2[j / 4 % 2 * 2] = add2(sum2[j / 4 % 2 * 2], pack2(ex2(y[0]), ex2(y[1])));
                            sum2[j / 4 % 2 * 2 + 1] = add2(sum2[j / 4 % 2 * 2 + 1], pack2(ex2(y[2]), ex2(y[3])));
                        }
                    };
                    // the next 32 columns are on their way while these are worked on
                    const uint32_t from = tmem_row + 128u * buf;
                    tc_ld32_nowait(from, v[0]);
                    tc_ld_wait_for(v[0]);
                    if (edge) {
                        const int chunks = (cols + 31) / 32;
                        for (int c = 0; c < chunks; ++c) {
                            chunk(std::true_type{}, c, v[0]);
                            if (c + 1 < chunks) { tc_ld32_nowait(from + 32u * (c + 1), v[0]); tc_ld_wait_for(v[0]); }
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (c < 3) tc_ld32_nowait(from + 32u * (c + 1), v[(c + 1) & 1]);
                            chunk(std::false_type{}, c, v[c & 1]);
                            if (c < 3) tc_ld_wait_for(v[(c + 1) & 1]);
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(s_empty + 16 * g + 8 * buf);
                }
                if (there && e < t.entries && ok) {
                    float x, y;
                    unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), x, y);
                    if (a.part_w) a.part_w[(((size_t)t.part * a.w.R + t.r) * a.w.nkv + t.kvh) * a.w.limit + e] = x + y;
                    else place(t)[e] = before + (x + y);
                }
            }
        } else {
            while (ok) {
                ok = next_item(t);
                if (!ok || t.n_m == 0) break;
                const bool both = t.n_m == 1;                        // both sides work on one tile
                const int tile = t.m0 + (both ? 0 : g), r = tile * a.tile_rows + row / group;
                const bool query = row < a.tile_rows * group && r < t.rows;
                const int sees = min(t.entries, t.start + r + 1);                       // entries that this lane's row sees
                const int first = min(t.entries, t.start + tile * a.tile_rows + 1);     // .. and the tile's first row
                float ref = -INFINITY, l = 0.f;
                for (int b = 0; b < t.n_b && ok; ++b) {
                    if (!mine_is(g, b)) continue;
                    const int buf = si & 1, k0 = (t.b0 + b * a.parts) * KT_TILE;
                    ok = mbar_wait_all(s_full + 16 * g + 8 * buf, (si >> 1) & 1, a.err, 77, &abort_flag);
                    if (!ok) break;
                    ++si;
                    tc_fence_after();
                    // 64 scores at a time under a reference that the first ones seen set: below 2^100 a sum is as good under
                    // any reference, above it the reference is raised.
                    if (__any_sync(0xffffffffu, query && k0 < sees)) {
                        const bool edge = k0 + KT_TILE > first;
                        uint32_t v[2][2][32];
                        const uint32_t from = tmem_row + 128u * buf;
                        tc_ld32_nowait(from, v[0][0]);
                        tc_ld32_nowait(from + 32u, v[0][1]);
                        tc_ld_wait_for(v[0][0]);
                        tc_ld_wait_for(v[0][1]);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (c == 0) { tc_ld32_nowait(from + 64u, v[1][0]); tc_ld32_nowait(from + 96u, v[1][1]); }
                            uint32_t (&x)[2][32] = v[c];
                            if (edge) {
#pragma unroll
                                for (int j = 0; j < 64; ++j)
                                    if (k0 + 64 * c + j >= sees) x[j >> 5][j & 31] = 0xff800000u;
                            }
                            auto pass = [&](float m) -> float {
                                uint64_t s2[4] = {0ull, 0ull, 0ull, 0ull};
                                const uint64_t nm2 = pack2(-m, -m);
#pragma unroll
                                for (int j = 0; j < 64; j += 2) {
                                    float y0, y1;
                                    unpack2(fma2(pack2(__uint_as_float(x[j >> 5][j & 31]), __uint_as_float(x[j >> 5][(j & 31) + 1])), scale2, nm2), y0, y1);
                                    s2[j / 2 % 4] = add2(s2[j / 2 % 4], pack2(ex2(y0), ex2(y1)));
                                }
                                float y0, y1;
                                unpack2(add2(add2(s2[0], s2[1]), add2(s2[2], s2[3])), y0, y1);
                                return y0 + y1;
                            };
                            float sum = 0.f;
                            bool raise = __any_sync(0xffffffffu, query && ref == -INFINITY);
                            if (!raise) {
                                sum = pass(ref == -INFINITY ? 0.f : ref);
                                raise = __any_sync(0xffffffffu, query && !(sum < 0x1p100f));
                            }
                            if (raise) {
                                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                                for (int j = 0; j < 64; ++j) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(x[j >> 5][j & 31]));
                                const float m = fmaxf(ref, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.w.scale_log2);
                                if (m > ref) { l *= ex2(ref - m); ref = m; }            // ref -inf: l is 0
                                sum = pass(ref == -INFINITY ? 0.f : ref);
                            }
                            l += sum;
                            if (c == 0) { tc_ld_wait_for(v[1][0]); tc_ld_wait_for(v[1][1]); }
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(s_empty + 16 * g + 8 * buf);
                }
                if (!ok) break;
                if (both) {                                          // side 1's result goes to side 0
                    if (g == 1) {
                        if (xi > 0) ok = mbar_wait_all(x_empty, (xi & 1) ^ 1, a.err, 79, &abort_flag);
                        if (!ok) break;
                        other_ml[row][0] = ref;
                        other_ml[row][1] = l;
                        mbar_arrive(x_full);
                    } else {
                        ok = mbar_wait_all(x_full, xi & 1, a.err, 80, &abort_flag);
                        if (!ok) break;
                        const float m = other_ml[row][0], n = fmaxf(ref, m), base_m = n == -INFINITY ? 0.f : n;
                        l = l * ex2(ref - base_m) + other_ml[row][1] * ex2(m - base_m);
                        ref = n;
                        mbar_arrive(x_empty);
                    }
                    ++xi;
                }
                if (query && !(both && g == 1)) {
                    const size_t at = (size_t)(t.row0 + r) * a.w.nh + t.kvh * group + row % group;
                    if (a.parts == 1) a.w.z[at] = l == 0.f ? INFINITY : ref + log2f(l);
                    else *reinterpret_cast<float2*>(a.part_ml + (at * a.parts + t.part) * 2) = make_float2(ref, l);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {                                                // give copies in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 9) {
        tc_fence_after();
        tmem_free(tmem, 512u);
    }
}

// z of every query of every request from its parts.
__global__ void __launch_bounds__(256) join_row_sums_kernel(const KtArgs a) {
    pdl_wait();
    pdl_trigger();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)a.w.T * a.w.nh) return;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + i * a.row_parts;
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < a.row_parts; ++p) {
        const float2 x = ml[p];
        const float n = fmaxf(m, x.x), ref = n == -INFINITY ? 0.f : n;
        l = l * ex2(m - ref) + x.y * ex2(x.x - ref);
        m = n;
    }
    a.w.z[i] = l == 0.f ? INFINITY : m + log2f(l);
}

// The weights from the second pass's parts, in the parts' order.  grid (entries / 256, nkv, R)
__global__ void __launch_bounds__(256) join_entry_sums_kernel(const KtArgs a) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y, e = blockIdx.x * 256 + threadIdx.x, slot = a.w.slots[r];
    int row0, rows, start, entries;
    rows_of(a.w, r, row0, rows, start, entries);
    if (e >= entries || slot < 0 || slot >= a.w.n_slots) return;
    float* w = a.w.weights + ((size_t)slot * a.w.nkv + kvh) * a.w.weights_ld + e;
    float sum = 0.f;
    for (int p = 0; p < a.parts; ++p) sum += a.part_w[(((size_t)p * a.w.R + r) * a.w.nkv + kvh) * a.w.limit + e];
    *w = (e < a.w.fresh[r] ? *w : 0.f) + sum;
}

// The queries as the tensor cores' kernel reads them: 64 columns of a head, heads, rows; a box of one kv head's and `rows` rows.
static int make_q_map(CUtensorMap* map, const void* q, int T, int q_stride, int nh, int d, int heads, int rows) {
    RgEncodeTiledFn fn = rg_encode_fn();
    if (!fn) return RG_ERR_UNSUPPORTED;
    cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)nh, (cuuint64_t)T}, strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)rows}, estr[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 20000 + (int)r;
}

static int join_rows(const KtArgs& a, cudaStream_t s) {
    if (a.parts == 1) return 0;
    return rg_launch(join_row_sums_kernel, dim3((unsigned)(((long long)a.w.T * a.w.nh + 255) / 256)), dim3(256), 0, s, 1, a);
}
static int join_entries(const KtArgs& a, int max_context, cudaStream_t s) {
    if (a.parts == 1) return 0;
    return rg_launch(join_entry_sums_kernel, dim3((max_context + 255) / 256, a.w.nkv, a.w.R), dim3(256), 0, s, 1, a);
}

template <int PIECES>
static int launch_key_weights_tc(KtArgs rows, KtArgs entries, int num_pages, int max_context, int sms, cudaStream_t s) {
    constexpr int smem = (2 * kt_a_stages(PIECES) + kt_b_stages(PIECES)) * KT_TILE * 128 * PIECES + 1024;
    const WeightArgs& w = rows.w;
    CUtensorMap qm, km;
    int e = make_q_map(&qm, w.q, w.T, w.q_stride, w.nh, w.d, w.nh / w.nkv, rows.tile_rows);
    if (e) return e;
    e = rg_make_map(&km, w.kv, (unsigned long long)num_pages * 2 * w.nkv * w.page_size, w.d, w.d, min(w.page_size, KT_TILE));
    if (e) return e;
    RG_ALLOW_SMEM((key_weights_tc_kernel<PIECES, false>), smem)
    RG_ALLOW_SMEM((key_weights_tc_kernel<PIECES, true>), smem)
    e = rg_launch(key_weights_tc_kernel<PIECES, false>, dim3(min(sms, rows.n_items)), dim3(KT_THREADS), smem, s, 1, qm, km, rows);
    if (!e) e = join_rows(rows, s);
    if (!e) e = rg_launch(key_weights_tc_kernel<PIECES, true>, dim3(min(sms, entries.n_items)), dim3(KT_THREADS), smem, s, 1, qm, km, entries);
    return e ? e : join_entries(entries, max_context, s);
}

template <typename A, bool VEC, int QI>
static int launch_key_weights_general(const KtArgs& rows, const KtArgs& entries, int max_rows, int max_context, cudaStream_t s) {
    const WeightArgs& w = rows.w;
    const size_t smem = kw_smem(w.d, 8 * QI);
    const long long q_tiles = ((long long)max_rows * (w.nh / w.nkv) + 8 * QI - 1) / (8 * QI), e_tiles = (max_context + KW_K - 1) / KW_K;
    if (q_tiles * rows.parts > 0x7fffffffll || e_tiles * entries.parts > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
    RG_ALLOW_SMEM((row_sums_general_kernel<A, VEC, QI>), kw_smem(256, 8 * QI))
    RG_ALLOW_SMEM((entry_sums_general_kernel<A, VEC, QI>), kw_smem(256, 8 * QI))
    int e = rg_launch(row_sums_general_kernel<A, VEC, QI>, dim3((unsigned)(q_tiles * rows.parts), w.nkv, w.R), dim3(KW_THREADS), smem, s, 1, rows);
    if (!e) e = join_rows(rows, s);
    if (!e)
        e = rg_launch(entry_sums_general_kernel<A, VEC, QI>, dim3((unsigned)(e_tiles * entries.parts), w.nkv, w.R), dim3(KW_THREADS), smem, s, 1,
                      entries);
    return e ? e : join_entries(entries, max_context, s);
}

// max_rows: the most rows of a request; max_context: the most entries a row sees.  Scratch: z [T, nh], part_ml [T, nh, row_parts,
// 2] where row_parts > 1 and part_w [entry_parts, R, nkv, max_context] where entry_parts > 1.
extern "C" int rg_prompt_key_weights(const void* q, int q_stride, const void* kv, int num_pages, int dtype, float* weights, int weights_ld,
                                     int n_slots, const int* slots, const int* block_table, int max_blocks, const int* cu_rows,
                                     const int* starts, const int* fresh, int R, int T, int nh, int nkv, int d, int page_size,
                                     float scale, int max_rows, int max_context, float* z, int row_parts, float* part_ml,
                                     int entry_parts, float* part_w, int tensor_cores, int sms, int* err, void* stream) {
    if (R <= 0 || T <= 0 || max_rows <= 0 || max_context <= 0) return 0;
    if (d < 1 || d > 256 || nkv < 1 || nh < nkv || nh % nkv || page_size < 1 || max_context > weights_ld || R > 65535 || nkv > 65535 ||
        (long long)max_rows * (nh / nkv) > 0x7fffff00ll || max_context > 0x7fffff00 || row_parts < 1 || entry_parts < 1)
        return RG_ERR_UNSUPPORTED;
    const WeightArgs a = {q, kv, block_table, cu_rows, starts, fresh, slots, weights, z, weights_ld, q_stride, max_blocks, n_slots, T, R,
                          nh, nkv, d, page_size, (int)min((long long)max_context, (long long)max_blocks * page_size),
                          scale * 1.4426950408889634f, max_rows};
    const cudaStream_t s = (cudaStream_t)stream;
    const int group = nh / nkv;
    KtArgs rows = {a, part_ml, nullptr, row_parts, row_parts}, entries = rows;
    entries.parts = entry_parts;
    entries.part_w = entry_parts > 1 ? part_w : nullptr;
    if (tensor_cores) {
        int shift = -1;
        for (int b = 3; b < 31; ++b) if (page_size == (1 << b)) shift = b;
        if (dtype != RG_DTYPE_BF16 || (d != 64 && d != 128) || group > KT_TILE || shift < 0 || q_stride % 8 || ((uintptr_t)q & 15) ||
            ((uintptr_t)kv & 15) || scale <= 0.f || (long long)num_pages * 2 * nkv * page_size > 0x7fffffffll)
            return RG_ERR_UNSUPPORTED;
        rows.err = entries.err = err;
        rows.page_shift = entries.page_shift = shift;
        rows.tile_rows = entries.tile_rows = KT_TILE / group;
        const long long q_tiles = (max_rows + rows.tile_rows - 1) / rows.tile_rows, e_tiles = (max_context + KT_TILE - 1) / KT_TILE;
        rows.blocks = (int)((q_tiles + 1) / 2);
        entries.blocks = (int)((e_tiles + 1) / 2);
        const long long n_rows = (long long)rows.blocks * R * nkv * row_parts, n_entries = (long long)entries.blocks * R * nkv * entry_parts;
        if (n_rows > 0x3fffffffll || n_entries > 0x3fffffffll) return RG_ERR_UNSUPPORTED;
        rows.n_items = (int)n_rows;
        entries.n_items = (int)n_entries;
        return d == 64 ? launch_key_weights_tc<1>(rows, entries, num_pages, max_context, sms, s)
                       : launch_key_weights_tc<2>(rows, entries, num_pages, max_context, sms, s);
    }
    const bool vec = d % 4 == 0 && q_stride % 4 == 0 && (((uintptr_t)q | (uintptr_t)kv) & (dtype == RG_DTYPE_F32 ? 15 : 7)) == 0;
#define RG_KW(A, V) { if (max_rows * group <= KW_FEW) return launch_key_weights_general<A, V, 2>(rows, entries, max_rows, max_context, s); \
    return launch_key_weights_general<A, V, 8>(rows, entries, max_rows, max_context, s); }
    if (dtype == RG_DTYPE_F32) { if (vec) RG_KW(float, true) RG_KW(float, false) }
    if (vec) RG_KW(bf16, true)
    RG_KW(bf16, false)
#undef RG_KW
}
