// Attention of single tokens in parts that are joined afterwards: behind prefixes that rows share (prefix_attention), and
// with the sum of the weights that every cached entry receives (weighed_attention).  attention_parts.cuh says how parts
// are cut and joined.
#include "attention_parts.cuh"
#include "mma.cuh"
#include "attention_prefix_tcgen05.cuh"
#include "attention_runs.cuh"

#define PG_THREADS 128
#define PG_Q 16                // queries of a block
#define PG_K 64                // entries of a tile
#define PG_LD (PG_K + 4)

// ---------------------------------------------------------------------------------------------------
// Any head size up to 256, any page size, 32-bit or bfloat16 storage, all arithmetic in 32-bit.
// Per tile of 64 entries: 2 queries x 4 entries of scores a thread, then a column of the output for all 16 queries a thread;
// DP = 32 or 64: as many threads share the columns, and PG_THREADS / DP groups of them share the tile's entries.  What bounds it is
// its arithmetic and the shared memory it reads from: 32-bit, 32 heads on 8 of 128, a prefix of 2,048 for 32 rows 157 us (7
// TFLOP/s), single tokens of 16 requests on 2,048 entries 232 us (1.2 TB/s); three heads of 32 on 63 entries 6.6 us, of which
// the launch is most.
// ---------------------------------------------------------------------------------------------------
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

// Where whole rows go: blocks that see all of a row's entries, or share them in a cluster, leave no parts.
struct RowsArgs {
    void* out;                   // [T, out_ld]
    float* weights;              // [n_slots, nkv, weights_ld]
    const int* slots;            // [T]
    long long weights_ld;
    int out_ld, n_slots, runs;   // runs: of 16 entries a block may have (its scores' place in shared memory)
    float decay;
};

__host__ __device__ inline int pg_row(int d) { return ((d + 3) & ~3) + 4; }   // floats a row in shared memory
__host__ __device__ inline int pg_stages(int d) { return d <= 128 ? 2 : 1; }   // tiles of K and V in shared memory: the next one is on its way

// WHOLE: a cluster takes all entries of a row, its prefix's and then its own, and leaves the output, and the weights where b has a
// place for them (their scores wait in a.scores).
template <typename A, int DP, bool VEC, bool WHOLE>
__global__ void __launch_bounds__(PG_THREADS) parts_general_kernel(const PartArgs a, const RowsArgs b) {
    extern __shared__ __align__(16) float smem[];
    constexpr int GROUPS = PG_THREADS / DP, COLS = DP == 128 ? 2 : 1;
    PartShare s;
    pdl_wait();
    pdl_trigger();
    int P = 0;
    const int* prefix_table = nullptr;
    int C = 1, rank = 0;
    if constexpr (WHOLE) {
        C = cg::this_cluster().num_blocks();
        rank = cg::this_cluster().block_rank();
        const int block = blockIdx.x / C, tile = block % a.own_tiles, tk = block / a.own_tiles;
        s.row0 = tk / a.nkv; s.kvh = tk % a.nkv; s.q0 = tile * PG_Q; s.nq = min(PG_Q, a.nh / a.nkv - s.q0);
        s.table = a.block_table + (size_t)s.row0 * a.max_blocks;
        s.e0 = 0; s.e1 = max(0, own_entries(a, s.row0));
        prefix_table = prefix_of(a, s.row0, P);
    } else if (!part_share(a, PG_Q, blockIdx.x, s)) return;
    const int d = a.d, ld = pg_row(d), group = a.nh / a.nkv, tid = threadIdx.x, stages = pg_stages(d);
    float* qs = smem;                                               // [16][ld]
    float* kv0 = qs + PG_Q * ld;                                    // [stages][K [64][ld], V [64][ld]]
    float* ps = kv0 + stages * 2 * PG_K * ld;                       // [16][PG_LD]
    float* al = ps + PG_Q * PG_LD;                                  // [16]
    __shared__ long long row_at[2][PG_K];                           // where the rows of a tile are in the cache, -1 behind its end
    const size_t page_elems = (size_t)2 * a.nkv * a.page_size * d, to_values = (size_t)a.nkv * a.page_size * d;
    const int prefix_tiles = (P + PG_K - 1) / PG_K, tiles = prefix_tiles + (s.e1 - s.e0 + PG_K - 1) / PG_K;
    const int per = (tiles + C - 1) / C, tile0 = min(tiles, rank * per), tile1 = min(tiles, tile0 + per);      // this block's
    // tile's first entry in its list, and how many entries of it there are
    auto tile_of = [&](int tile, int& e0) -> int {
        const bool shared = tile < prefix_tiles;                    // entries of the prefix
        e0 = shared ? tile * PG_K : s.e0 + (tile - prefix_tiles) * PG_K;
        return min(PG_K, (shared ? P : s.e1) - e0);
    };
    auto look_up = [&](int tile) -> long long {                     // threads 0 .. 63: a row each
        int e0;
        const int n = tile < tile1 ? tile_of(tile, e0) : 0;
        if (tid >= n) return -1;
        const int e = e0 + tid;
        return (long long)((tile < prefix_tiles ? prefix_table : s.table)[e / a.page_size]) * (long long)page_elems +
               ((long long)s.kvh * a.page_size + e % a.page_size) * d;
    };
    // a thread's pieces of a tile: every 128th
    const int pieces = VEC ? d / 4 : d, row_first = tid / pieces, piece_first = tid - row_first * pieces, row_step = PG_THREADS / pieces,
              piece_step = PG_THREADS - row_step * pieces;
    auto request = [&](int tile, float* ks) {                       // rows behind the end are zeros
        constexpr int W = VEC ? 4 : 1;
        float* vs = ks + PG_K * ld;
        for (int row = row_first, p = piece_first; row < PG_K; p += piece_step, row += row_step) {
            if (p >= pieces) { p -= pieces; if (++row >= PG_K) break; }
            const int c = p * W;
            const long long at = row_at[tile & 1][row];
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
            for (int i = tid; i < PG_K * (ld - d); i += PG_THREADS) ks[i / (ld - d) * ld + d + i % (ld - d)] = 0.f;
        rgmma::cp_async_commit();
    };
    if (tid < PG_K) { row_at[tile0 & 1][tid] = look_up(tile0); row_at[(tile0 + 1) & 1][tid] = look_up(tile0 + 1); }
    for (int i = tid; i < PG_Q * ld; i += PG_THREADS) {
        const int row = i / ld, c = i - row * ld, qi = s.q0 + row;
        float v = 0.f;
        if (row < s.nq && c < d)
            v = to_f32(((const A*)a.q)[(size_t)(s.row0 + qi / group) * a.q_stride + (s.kvh * group + qi % group) * d + c]) * a.scale_log2;
        qs[i] = v;
    }
    const int qa = tid >> 4, ka = tid & 15;                         // scores: queries 2 qa, 2 qa + 1; entries ka + 16 j
    float* keep[2];                                                 // where their scores go
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int qi = s.q0 + 2 * qa + i;
        keep[i] = a.scores && 2 * qa + i < s.nq ? a.scores + ((size_t)(s.row0 + qi / group) * a.nh + s.kvh * group + qi % group) * a.score_ld + ka : nullptr;
    }
    const int col = tid % DP, part = tid / DP;                      // output: column(s) col (+ 128), entries part + GROUPS j
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float acc[COLS][PG_Q];
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int i = 0; i < PG_Q; ++i) acc[c][i] = 0.f;
    __syncthreads();
    if (stages == 2 && tile0 < tile1) request(tile0, kv0 + (tile0 & 1) * 2 * PG_K * ld);
    for (int tile = tile0; tile < tile1; ++tile) {
        int e0;
        const bool shared = tile < prefix_tiles;
        const int n = tile_of(tile, e0);
        float* ks = kv0 + (stages == 2 ? (tile & 1) * 2 * PG_K * ld : 0);
        const float* vs = ks + PG_K * ld;
        if (stages == 1) {
            __syncthreads();                                        // the last tile's values are read
            request(tile, ks);
        }
        rgmma::cp_async_wait<0>();
        __syncthreads();                                            // the tile is there; with two stages the last one is read
        if (stages == 2 && tile + 1 < tile1) request(tile + 1, kv0 + ((tile + 1) & 1) * 2 * PG_K * ld);
        const long long at_next = tid < PG_K ? look_up(tile + 2) : -1;
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
                if (ka + 16 * j >= n) sc[i][j] = -INFINITY;
                else if (keep[i] && !shared) keep[i][e0 + 16 * j] = sc[i][j];
                mx = fmaxf(mx, sc[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(m[i], mx), ms = mn == -INFINITY ? 0.f : mn, f = exp2f(m[i] - ms);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(sc[i][j] - ms);
                ps[(2 * qa + i) * PG_LD + ka + 16 * j] = p;
                sum += p;
            }
            l[i] = l[i] * f + sum;                                  // this thread's entries; added up at the end
            m[i] = mn;
            if (ka == 0) al[2 * qa + i] = f;
        }
        __syncthreads();
        if (tid < PG_K) row_at[tile & 1][tid] = at_next;            // requested from after the next barrier
#pragma unroll
        for (int i = 0; i < PG_Q; ++i) {
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
            for (int i = 0; i < PG_Q; ++i) {
                const float4 p4 = *reinterpret_cast<const float4*>(ps + i * PG_LD + e);
#pragma unroll
                for (int c = 0; c < COLS; ++c) {
                    acc[c][i] += p4.x * v[c][0]; acc[c][i] += p4.y * v[c][1];
                    acc[c][i] += p4.z * v[c][2]; acc[c][i] += p4.w * v[c][3];
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
    }
    if constexpr (GROUPS > 1) {                                     // the groups' sums, added in their order
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PG_Q; ++i) kv0[i * PG_THREADS + tid] = acc[0][i];
        __syncthreads();
        if (part == 0) {
#pragma unroll
            for (int i = 0; i < PG_Q; ++i)
                for (int g = 1; g < GROUPS; ++g) acc[0][i] += kv0[i * PG_THREADS + g * DP + col];
        }
    }
    if constexpr (WHOLE) {
        __shared__ float fin_ml[PG_Q][2], row_ml[PG_Q][2];          // this block's M and L; the row's M and 1 / L
        cg::cluster_group cluster = cg::this_cluster();
        float* fin = kv0;                                           // [16][d]
        __syncthreads();                                            // the last tile and the groups' sums are read
        if (part == 0) {
#pragma unroll
            for (int i = 0; i < PG_Q; ++i)
                if (i < s.nq)
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
                        if (col + DP * c < d) fin[i * d + col + DP * c] = acc[c][i];
        }
        if (ka == 0)
#pragma unroll
            for (int i = 0; i < 2; ++i) { fin_ml[2 * qa + i][0] = m[i]; fin_ml[2 * qa + i][1] = l[i]; }
        cluster.sync();                                             // every block's result is in place
        if (tid < s.nq) join_cluster_ml(cluster, &fin_ml[0][0], tid, row_ml[tid][0], row_ml[tid][1]);
        __syncthreads();
        const int h0 = s.kvh * group + s.q0;
        for (int idx = rank * PG_THREADS + tid; idx < s.nq * d; idx += C * PG_THREADS) {
            const int r = idx / d, c = idx - r * d;
            float sum = 0.f;
            for (int k = 0; k < C; ++k)
                sum += exp2f(cluster.map_shared_rank(&fin_ml[0][0], k)[r * 2] - row_ml[r][0]) * cluster.map_shared_rank(fin, k)[r * d + c];
            ((A*)b.out)[(size_t)s.row0 * b.out_ld + (h0 + r) * d + c] = from_f32<A>(sum * row_ml[r][1]);
        }
        const int slot = b.weights ? b.slots[s.row0] : -1;
        if (slot >= 0 && slot < b.n_slots) {
            float* to = b.weights + ((size_t)slot * a.nkv + s.kvh) * b.weights_ld;
            const int first = max(0, tile0 - prefix_tiles) * PG_K, last = min(s.e1, (tile1 - prefix_tiles) * PG_K);   // own entries of this block
            const int newest = a.positions[s.row0];                   // behind what there is room for: none of them is new
            for (int e = first + tid; e < last; e += PG_THREADS) {
                const float* sc = a.scores + ((size_t)s.row0 * a.nh + h0) * a.score_ld + e;
                float sum = 0.f;
                for (int i = 0; i < s.nq; ++i) sum += exp2f(sc[(size_t)i * a.score_ld] - row_ml[i][0]) * row_ml[i][1];
                to[e] = (e == newest ? 0.f : b.decay * to[e]) + sum;
            }
        }
        cluster.sync();                                             // nobody leaves while its results are being read
        return;
    }
    const int slots = a.prefix_parts + a.own_parts;
    auto place = [&](int row) -> size_t {
        const int qi = s.q0 + row;
        return ((size_t)(s.row0 + qi / group) * a.nh + s.kvh * group + qi % group) * slots + s.slot;
    };
    if (part == 0) {
#pragma unroll
        for (int i = 0; i < PG_Q; ++i)
            if (i < s.nq)
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (col + DP * c < d) a.part_o[place(i) * d + col + DP * c] = acc[c][i];
    }
    if (ka == 0)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (2 * qa + i < s.nq) {
                a.part_ml[place(2 * qa + i) * 2] = m[i];
                a.part_ml[place(2 * qa + i) * 2 + 1] = l[i];
            }
}

// ---------------------------------------------------------------------------------------------------
// bfloat16, head sizes 64, 128, 192 and 256, pages of 8 tokens or a larger power of two: mma.sync m16n8k16 on tiles that TMA
// brings.  What bounds it is memory: every entry's K and V are read once for up to 16 queries.  64 requests on 4,096 entries each,
// 32 heads on 8, with their weights: 190 us at head size 128 (5.7 TB/s, 89 % of what a copy reaches), 112 at 64 (5.0 TB/s); on 1 to
// 4,096 entries at head size 128 104 us, some 10 of which are the tail of unequal blocks and the kernel that joins.  (Blocks that
// stay and take several parts each: 202 to 214 us for the equal lists.)  One request on 32,768 entries: 33 us.
//
// A block is four warps that share nothing until they join at the end.  A warp takes every fourth run of 16 entries: one TMA
// box of K and V together (a four-dimensional map: 64 columns, rows, 64-column pieces of the head, K and V; pages of 8 take
// two boxes) into a ring of its own, refilled by the warp itself as soon as it has read a stage: no barrier between warps,
// no copy instructions beside one a run.  The 128-byte swizzle keeps ldmatrix free of conflicts.
// ---------------------------------------------------------------------------------------------------
template <int PIECES, bool BRIEF>
__global__ void __launch_bounds__(PM_THREADS, pm_blocks(PIECES, BRIEF))
parts_mma_kernel(const __grid_constant__ CUtensorMap kv_map, const PartArgs a, int* err) {
    constexpr int D = 64 * PIECES, STAGES = pm_stages(PIECES, BRIEF), STAGE = pm_stage_bytes(PIECES);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[4 * STAGES];
    __shared__ float ml[4][PM_Q][2];
    __shared__ int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t first_stage = (smem_addr(smem_raw) + 1023u) & ~1023u, base = first_stage + (uint32_t)(warp * STAGES * STAGE);
    const uint32_t bar0 = smem_addr(bars) + (uint32_t)(8 * STAGES * warp);
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        fence_barrier_init();
    }
    __syncthreads();
    // beside: the launch before this one is prefix_tc_kernel for the same rows, whose blocks have all waited for what came
    // before them; it leaves its own parts.  What comes behind this kernel waits for both: the last block waits at its end.
    if (!a.beside) pdl_wait();
    pdl_trigger();
    PartShare sh;
    const bool closes = a.beside && blockIdx.x == gridDim.x - 1;
    if (!part_share(a, PM_Q, blockIdx.x, sh)) {
        if (closes) pdl_wait();
        return;
    }
    const int group = a.nh / a.nkv;
    const int n_runs = (sh.e1 - sh.e0 + 15) >> 4, mine = n_runs > warp ? (n_runs - warp + 3) >> 2 : 0;
    // Page ids of this warp's next 32 runs, one a lane (of both halves of a run where pages hold 8).
    const int box_shift = a.page_shift < 4 ? 3 : 4;
    int page_a = 0, page_b = 0;
    auto entry_of = [&](int i) -> int { return sh.e0 + (warp + 4 * i) * 16; };
    auto issue = [&](int i) {                                         // the whole warp: run i of this warp
        if ((i & 31) == 0) {
            const int e = entry_of(i + lane);
            page_a = e < sh.e1 ? sh.table[e >> a.page_shift] : 0;
            if (box_shift == 3) page_b = e + 8 < sh.e1 ? sh.table[(e + 8) >> a.page_shift] : page_a;   // no such entry: any page
        }
        const int pa = __shfl_sync(0xffffffffu, page_a, i & 31), pb = __shfl_sync(0xffffffffu, page_b, i & 31);
        if (lane == 0) load_run(&kv_map, a.nkv, a.page_size, base + (i % STAGES) * STAGE, bar0 + 8 * (i % STAGES), STAGE, box_shift, pa, pb, sh.kvh, entry_of(i));
        __syncwarp();
    };
    for (int i = 0; i < min(STAGES, mine); ++i) issue(i);

    MmaQueries<PIECES> w;
    w.init(lane, box_shift);
    const int qa = sh.q0 + w.g, qb = qa + 8;
    auto head_of = [&](int qi) -> int { return sh.kvh * group + qi % group; };
    auto row_of = [&](int qi) -> int { return sh.row0 + qi / group; };
    const bool has_a = w.g < sh.nq, has_b = w.g + 8 < sh.nq;
    w.queries(has_a ? (const bf16*)a.q + (size_t)row_of(qa) * a.q_stride + head_of(qa) * D : nullptr,
              has_b ? (const bf16*)a.q + (size_t)row_of(qb) * a.q_stride + head_of(qb) * D : nullptr);
    float *score_a = nullptr, *score_b = nullptr;
    if (a.scores) {
        if (has_a) score_a = a.scores + ((size_t)row_of(qa) * a.nh + head_of(qa)) * a.score_ld + 2 * w.tq;
        if (has_b) score_b = a.scores + ((size_t)row_of(qb) * a.nh + head_of(qb)) * a.score_ld + 2 * w.tq;
    }
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
        const int s = i % STAGES, e = entry_of(i);
        ok = mbar_wait_all(bar0 + 8 * s, (i / STAGES) & 1, err, 61, &abort_flag);
        if (!ok) break;
        w.step(base + s * STAGE, sh.e1 - e, a.scale_log2, [&](const float (&v)[8]) {
            if (score_a) {
                *reinterpret_cast<float2*>(score_a + e) = make_float2(v[0], v[1]);
                *reinterpret_cast<float2*>(score_a + e + 8) = make_float2(v[2], v[3]);
            }
            if (score_b) {
                *reinterpret_cast<float2*>(score_b + e) = make_float2(v[4], v[5]);
                *reinterpret_cast<float2*>(score_b + e + 8) = make_float2(v[6], v[7]);
            }
        });
        if (i + STAGES < mine) issue(i + STAGES);
    }
    if (!ok || abort_flag)                                            // give copies in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    // the four warps' results, through the stages' memory (every copy has landed and been read)
    __syncthreads();
    float* all = reinterpret_cast<float*>(smem_raw + (first_stage - smem_addr(smem_raw)));   // [4][16][D]
    w.leave(all + warp * PM_Q * D, ml[warp]);
    __syncthreads();
    const int slots = a.prefix_parts + a.own_parts;
    for (int idx = threadIdx.x; idx < sh.nq * (D / 4); idx += PM_THREADS) {
        const int r = idx / (D / 4), c = idx % (D / 4) * 4, qi = sh.q0 + r;
        float M, L;
        const float4 sum = join_warps<D>(all, ml, r, c, M, L);
        const size_t place = ((size_t)row_of(qi) * a.nh + head_of(qi)) * slots + sh.slot;
        *reinterpret_cast<float4*>(a.part_o + place * D + c) = sum;
        if (c == 0) *reinterpret_cast<float2*>(a.part_ml + place * 2) = make_float2(M, L);
    }
    if (closes) pdl_wait();
}

// ---------------------------------------------------------------------------------------------------
// Few rows, in one launch: a cluster takes a row and up to 16 heads of a kv head and cuts the row's entries (its prefix's, then
// its own) among its blocks, which join through each other's shared memory.  A prefix is then read once for every row, out
// of L2; what is saved is the second launch and the parts' trip through memory.  With WEIGH the scores stay in shared memory
// until the row's sums are known, and the entries' weights are written by the block that read them.  What bounds it is the launch,
// one trip to memory for the table and one for the entries: one request on 1,024 entries at head size 64 with weights 5.7 us
// (7.8 in parts that a second kernel joins); 4 rows on 1,024 shared and 64 own entries at 128 8.7 (10.0 in parts).
// grid (T clusters, nkv x tiles of heads)
// ---------------------------------------------------------------------------------------------------
template <int PIECES, bool WEIGH, bool BRIEF>
__global__ void __launch_bounds__(PM_THREADS, pm_blocks(PIECES, BRIEF))
rows_mma_kernel(const __grid_constant__ CUtensorMap kv_map, const PartArgs a, const RowsArgs b, int* err) {
    constexpr int D = 64 * PIECES, STAGES = pm_stages(PIECES, BRIEF), STAGE = pm_stage_bytes(PIECES);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t bars[4 * STAGES];
    __shared__ float ml[4][PM_Q][2], fin_ml[PM_Q][2], row_ml[PM_Q][2];
    __shared__ int abort_flag;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t first_stage = (smem_addr(smem_raw) + 1023u) & ~1023u, base = first_stage + (uint32_t)(warp * STAGES * STAGE);
    const uint32_t bar0 = smem_addr(bars) + (uint32_t)(8 * STAGES * warp);
    float* all = reinterpret_cast<float*>(smem_raw + (first_stage - smem_addr(smem_raw)));   // [4][16][D], then the block's [16][D]
    float* fin = all + 4 * PM_Q * D;
    float* scores = all + 4 * STAGES * STAGE / 4;                     // [heads][ld]
    const int ld = b.runs * 16 + 8;
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        fence_barrier_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x / C, group = a.nh / a.nkv, kvh = blockIdx.y / a.own_tiles, q0 = blockIdx.y % a.own_tiles * PM_Q;
    const int nq = min(PM_Q, group - q0), h0 = kvh * group + q0;
    const int newest = a.positions[t];                                // asked for before the groups are looked at
    int P = 0;
    const int* prefix_table = prefix_of(a, t, P);
    const int own = max(0, min(newest + 1, a.own_limit)), prefix_runs = (P + 15) >> 4, total = prefix_runs + ((own + 15) >> 4);
    const int per = (total + C - 1) / C, first = min(total, rank * per), last = min(total, first + per);
    const int n_runs = last - first, mine = n_runs > warp ? (n_runs - warp + 3) >> 2 : 0;
    const int* own_table = a.block_table + (size_t)t * a.max_blocks;
    const int box_shift = a.page_shift < 4 ? 3 : 4;
    int page_a = 0, page_b = 0;
    // run i of this warp: its first entry in the list that it is in, and how many entries that list has from there on
    auto place_of = [&](int i, int& e, int& n) -> const int* {
        const int run = first + warp + 4 * i;
        const bool shared = run < prefix_runs;
        e = (shared ? run : run - prefix_runs) * 16;
        n = (shared ? P : own) - e;
        return shared ? prefix_table : own_table;
    };
    auto issue = [&](int i) {
        int e, n;
        if ((i & 31) == 0) {
            const int* table = place_of(i + lane, e, n);
            const bool there = i + lane < mine;
            page_a = there ? table[e >> a.page_shift] : 0;
            if (box_shift == 3) page_b = there && n > 8 ? table[(e + 8) >> a.page_shift] : page_a;       // no such entry: any page
        }
        const int pa = __shfl_sync(0xffffffffu, page_a, i & 31), pb = __shfl_sync(0xffffffffu, page_b, i & 31);
        place_of(i, e, n);
        if (lane == 0) load_run(&kv_map, a.nkv, a.page_size, base + (i % STAGES) * STAGE, bar0 + 8 * (i % STAGES), STAGE, box_shift, pa, pb, kvh, e);
        __syncwarp();
    };
    for (int i = 0; i < min(STAGES, mine); ++i) issue(i);
    MmaQueries<PIECES> w;
    w.init(lane, box_shift);
    const bool has_a = w.g < nq, has_b = w.g + 8 < nq;
    const bf16* q = (const bf16*)a.q + (size_t)t * a.q_stride + (size_t)h0 * D;
    w.queries(has_a ? q + w.g * D : nullptr, has_b ? q + (w.g + 8) * D : nullptr);
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
        const int s = i % STAGES;
        int e, n;
        place_of(i, e, n);
        ok = mbar_wait_all(bar0 + 8 * s, (i / STAGES) & 1, err, 62, &abort_flag);
        if (!ok) break;
        w.step(base + s * STAGE, n, a.scale_log2, [&](const float (&v)[8]) {
            if constexpr (WEIGH) {
                float* to = scores + w.g * ld + (warp + 4 * i) * 16 + 2 * w.tq;
                if (has_a) {
                    *reinterpret_cast<float2*>(to) = make_float2(v[0], v[1]);
                    *reinterpret_cast<float2*>(to + 8) = make_float2(v[2], v[3]);
                }
                if (has_b) {
                    *reinterpret_cast<float2*>(to + 8 * ld) = make_float2(v[4], v[5]);
                    *reinterpret_cast<float2*>(to + 8 * ld + 8) = make_float2(v[6], v[7]);
                }
            }
        });
        if (i + STAGES < mine) issue(i + STAGES);
    }
    if (!ok || abort_flag)                                            // give copies in flight time to land
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
    w.leave(all + warp * PM_Q * D, ml[warp]);
    __syncthreads();
    for (int idx = threadIdx.x; idx < nq * (D / 4); idx += PM_THREADS) {
        const int r = idx / (D / 4), c = idx % (D / 4) * 4;
        float M, L;
        *reinterpret_cast<float4*>(fin + r * D + c) = join_warps<D>(all, ml, r, c, M, L);
        if (c == 0) { fin_ml[r][0] = M; fin_ml[r][1] = L; }
    }
    cluster.sync();                                                   // every block's result is in place
    if (threadIdx.x < nq) join_cluster_ml(cluster, &fin_ml[0][0], threadIdx.x, row_ml[threadIdx.x][0], row_ml[threadIdx.x][1]);
    __syncthreads();
    for (int idx = rank * PM_THREADS + threadIdx.x; idx < nq * (D / 4); idx += C * PM_THREADS) {
        const int r = idx / (D / 4), c = idx % (D / 4) * 4;
        float4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < C; ++k) {
            const float f = ex2(cluster.map_shared_rank(&fin_ml[0][0], k)[r * 2] - row_ml[r][0]) * row_ml[r][1];
            const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(fin, k) + r * D + c);
            sum.x += f * x.x; sum.y += f * x.y; sum.z += f * x.z; sum.w += f * x.w;
        }
        bf16* to = (bf16*)b.out + (size_t)t * b.out_ld + (h0 + r) * D + c;
        to[0] = __float2bfloat16_rn(sum.x); to[1] = __float2bfloat16_rn(sum.y);
        to[2] = __float2bfloat16_rn(sum.z); to[3] = __float2bfloat16_rn(sum.w);
    }
    if constexpr (WEIGH) {
        const int slot = b.slots[t];
        if (slot >= 0 && slot < b.n_slots) {
            float* to = b.weights + ((size_t)slot * a.nkv + kvh) * b.weights_ld;
            for (int i = threadIdx.x; i < n_runs * 16; i += PM_THREADS) {
                const int e = first * 16 + i;
                if (e >= own) break;
                const float before = e == newest ? 0.f : b.decay * to[e];   // newest behind what there is room for: none
                float sum = 0.f;
                for (int r = 0; r < nq; ++r) sum += ex2(scores[r * ld + i] - row_ml[r][0]) * row_ml[r][1];
                to[e] = before + sum;
            }
        }
    }
    cluster.sync();                                                   // nobody leaves while its results are being read
}

// ---------------------------------------------------------------------------------------------------
// Joining the parts of a row and head, and adding up the weights of a row's entries over the heads of a kv head.  Short kernels
// that are bound by their trips to memory: 64 rows of 32 heads in parts of 128 numbers 9.7 us from a cold cache, 64 requests'
// outputs and weights of 1 to 4,096 entries from 32 heads' scores 14 (25 MB read).
// ---------------------------------------------------------------------------------------------------
#define JOIN_THREADS 128

// What this row's softmax came to, from its parts: M and L of head h, by a whole warp (same result in every lane).
__device__ __forceinline__ void join_ml(const PartArgs& a, int t, int h, int n_prefix, int n_own, float& M, float& L) {
    const int slots = a.prefix_parts + a.own_parts, lane = threadIdx.x & 31, n = n_prefix + n_own;
    const float* ml = a.part_ml + ((size_t)t * a.nh + h) * slots * 2;
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < n; i += 32) {
        const int slot = i < n_prefix ? i : a.prefix_parts + i - n_prefix;
        const float mi = ml[slot * 2], mn = fmaxf(m, mi), ms = mn == -INFINITY ? 0.f : mn;
        l = l * exp2f(m - ms) + ml[slot * 2 + 1] * exp2f(mi - ms);
        m = mn;
    }
    M = warp_max(m);
    const float ms = M == -INFINITY ? 0.f : M;
    L = warp_sum(l * exp2f(m - ms));
    M = ms;
}

// The output of row t and head h.  The block's four warps take every fourth part, four columns a lane; their sums are added in
// their order.
#define JOIN_PARTS 512            // factors kept at a time
template <typename A>
__device__ __forceinline__ void join_row(const PartArgs& a, int t, int h, A* __restrict__ out, int out_ld) {
    __shared__ float factor[JOIN_PARTS];
    __shared__ float4 sums[JOIN_THREADS / 32][64];
    const int slots = a.prefix_parts + a.own_parts, d = a.d, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int position = a.positions[t];                              // asked for before the groups are looked at
    const int n_prefix = a.prefix_parts ? prefix_parts_of(a, t) : 0, n = n_prefix + own_parts_at(a, position);
    float M, L;
    join_ml(a, t, h, n_prefix, n - n_prefix, M, L);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const size_t base = ((size_t)t * a.nh + h) * slots;
    auto slot_of = [&](int i) -> size_t { return base + (i < n_prefix ? i : a.prefix_parts + i - n_prefix); };
    const bool quads = d % 4 == 0;
    float4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int i0 = 0; i0 < n; i0 += JOIN_PARTS) {
        const int m = min(JOIN_PARTS, n - i0);
        __syncthreads();
        for (int i = threadIdx.x; i < m; i += JOIN_THREADS) factor[i] = exp2f(a.part_ml[slot_of(i0 + i) * 2] - M) * inv;
        __syncthreads();
#pragma unroll 4
        for (int i = warp; i < m; i += JOIN_THREADS / 32) {
            const float f = factor[i];
            const float* from = a.part_o + slot_of(i0 + i) * d;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = 4 * lane + 128 * k;
                if (c >= d) continue;
                float4 x = {0.f, 0.f, 0.f, 0.f};
                if (quads) x = *reinterpret_cast<const float4*>(from + c);
                else { x.x = from[c]; if (c + 1 < d) x.y = from[c + 1]; if (c + 2 < d) x.z = from[c + 2]; if (c + 3 < d) x.w = from[c + 3]; }
                acc[k].x += f * x.x; acc[k].y += f * x.y; acc[k].z += f * x.z; acc[k].w += f * x.w;
            }
        }
    }
    sums[warp][lane] = acc[0];
    sums[warp][lane + 32] = acc[1];
    __syncthreads();
    A* to = out + (size_t)t * out_ld + h * d;
    for (int c = threadIdx.x; c < d; c += JOIN_THREADS) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < JOIN_THREADS / 32; ++w) v += reinterpret_cast<const float*>(&sums[w][0])[c];
        to[c] = from_f32<A>(v);
    }
}

// The same by one warp, parts in their order, where there are up to 32 of them: a part's factor a lane.
template <typename A>
__device__ __forceinline__ void join_row_warp(const PartArgs& a, int t, int h, A* __restrict__ out, int out_ld) {
    const int slots = a.prefix_parts + a.own_parts, d = a.d, lane = threadIdx.x & 31;
    const int position = a.positions[t];                              // asked for before the groups are looked at
    const int n_prefix = a.prefix_parts ? prefix_parts_of(a, t) : 0, n = n_prefix + own_parts_at(a, position);
    const size_t base = ((size_t)t * a.nh + h) * slots;
    const int slot = lane < n_prefix ? lane : a.prefix_parts + lane - n_prefix;
    float2 ml = {-INFINITY, 0.f};
    if (lane < n) ml = *reinterpret_cast<const float2*>(a.part_ml + (base + slot) * 2);
    const float M = warp_max(ml.x), e = exp2f(ml.x - (M == -INFINITY ? 0.f : M)), L = warp_sum(ml.y * e);
    const float factor = L == 0.f ? 0.f : e / L;
    A* to = out + (size_t)t * out_ld + h * d;
    for (int c0 = 0; c0 < d; c0 += 128) {
        const int c = c0 + 4 * lane;
        float4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float f = __shfl_sync(0xffffffffu, factor, i);
            const float* from = a.part_o + (base + (i < n_prefix ? i : a.prefix_parts + i - n_prefix)) * d + c;
            float4 x = {0.f, 0.f, 0.f, 0.f};
            if (d % 4 == 0) { if (c < d) x = *reinterpret_cast<const float4*>(from); }
            else { if (c < d) x.x = from[0]; if (c + 1 < d) x.y = from[1]; if (c + 2 < d) x.z = from[2]; if (c + 3 < d) x.w = from[3]; }
            acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
        }
        if (c < d) to[c] = from_f32<A>(acc.x);
        if (c + 1 < d) to[c + 1] = from_f32<A>(acc.y);
        if (c + 2 < d) to[c + 2] = from_f32<A>(acc.z);
        if (c + 3 < d) to[c + 3] = from_f32<A>(acc.w);
    }
}
// Rows and heads of a block: one, or one a warp where there are enough to fill the GPU and few parts (211 rows of 32 heads in five
// parts: 19 us with one a block, bound by instructions).
static int join_heads(const PartArgs& a) {
    return a.prefix_parts + a.own_parts <= 32 && (long long)a.T * a.nh >= 592 ? JOIN_THREADS / 32 : 1;
}
static unsigned join_blocks(const PartArgs& a) { return (unsigned)(((long long)a.T * a.nh + join_heads(a) - 1) / join_heads(a)); }
template <typename A>
__device__ __forceinline__ void join_block(const PartArgs& a, int b, int heads, A* __restrict__ out, int out_ld) {
    const int i = heads == 1 ? b : b * heads + (int)(threadIdx.x >> 5), t = i / a.nh, h = i % a.nh;
    if (heads == 1) join_row(a, t, h, out, out_ld);
    else if (t < a.T) join_row_warp(a, t, h, out, out_ld);
}

template <typename A>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const PartArgs a, int heads, A* __restrict__ out, int out_ld) {
    pdl_wait();
    pdl_trigger();
    join_block(a, blockIdx.x, heads, out, out_ld);
}

// The first `joins` blocks join rows and heads; the others add up the weights of 512 entries of a row and kv head, four a thread:
//   w[e] = decay w[e] + sum_h 2^(s_h(e) - M_h) / L_h,   w[positions[t]], the newest entry's, not read
#define WEIGH_CHUNK (4 * JOIN_THREADS)
#define WEIGH_HEADS 64
template <typename A>
__global__ void __launch_bounds__(JOIN_THREADS) weigh_kernel(const PartArgs a, int joins, int heads, A* __restrict__ out, int out_ld,
                                                             float* __restrict__ weights, long long weights_ld, int n_slots,
                                                             const int* __restrict__ slots, int chunks, float decay) {
    pdl_wait();
    pdl_trigger();
    int b = blockIdx.x;
    if (b < joins) { join_block(a, b, heads, out, out_ld); return; }
    b -= joins;
    const int chunk = b % chunks, kvh = b / chunks % a.nkv, t = b / chunks / a.nkv, group = a.nh / a.nkv;
    const int n = own_entries(a, t), newest = a.positions[t], e = chunk * WEIGH_CHUNK + 4 * threadIdx.x, slot = slots[t];
    if (chunk * WEIGH_CHUNK >= n || slot < 0 || slot >= n_slots) return;
    __shared__ float sM[WEIGH_HEADS], sI[WEIGH_HEADS];
    const int n_own = own_parts_of(a, t), warp = threadIdx.x >> 5;
    float* w = weights + ((size_t)slot * a.nkv + kvh) * weights_ld;
    float before[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) before[j] = e + j < n && e + j != newest ? decay * w[e + j] : 0.f;
    for (int g0 = 0; g0 < group; g0 += WEIGH_HEADS) {                // heads of a kv head, so many at a time
        const int some = min(group - g0, WEIGH_HEADS);
        __syncthreads();
        for (int g = warp; g < some; g += JOIN_THREADS / 32) {
            float M, L;
            join_ml(a, t, kvh * group + g0 + g, 0, n_own, M, L);
            if ((threadIdx.x & 31) == 0) { sM[g] = M; sI[g] = L == 0.f ? 0.f : 1.f / L; }
        }
        __syncthreads();
        if (e >= n) continue;
        const float* sc = a.scores + ((size_t)t * a.nh + kvh * group + g0) * a.score_ld + e;   // rows of whole 64 entries
#pragma unroll 4
        for (int g = 0; g < some; ++g) {
            const float4 s = *reinterpret_cast<const float4*>(sc + (size_t)g * a.score_ld);
            sum[0] += exp2f(s.x - sM[g]) * sI[g]; sum[1] += exp2f(s.y - sM[g]) * sI[g];
            sum[2] += exp2f(s.z - sM[g]) * sI[g]; sum[3] += exp2f(s.w - sM[g]) * sI[g];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (e + j < n) w[e + j] = before[j] + sum[j];
}

// ---------------------------------------------------------------------------------------------------
static size_t pg_smem(int d) { return (size_t)((PG_Q + pg_stages(d) * 2 * PG_K) * pg_row(d) + PG_Q * PG_LD + PG_Q) * sizeof(float); }

// whole: rows that go to their places, a cluster of blocks each (and tile of heads).
static int launch_parts_general(const PartArgs& a, int dtype, cudaStream_t s, const RowsArgs* whole = nullptr, int cluster = 1) {
    const long long blocks = whole ? (long long)a.T * a.nkv * a.own_tiles * cluster : part_blocks(a);
    if (blocks > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
    if (blocks == 0) return 0;
    const size_t smem = pg_smem(a.d);
    const bool vec = a.d % 4 == 0 && (((uintptr_t)a.kv) & (dtype == RG_DTYPE_F32 ? 15 : 7)) == 0;
    const RowsArgs b = whole ? *whole : RowsArgs{};
#define RG_PG_(A, DP, VEC, W) { RG_ALLOW_SMEM((parts_general_kernel<A, DP, VEC, W>), 160 * 1024) \
    return rg_launch(parts_general_kernel<A, DP, VEC, W>, dim3((unsigned)blocks), dim3(PG_THREADS), smem, s, cluster, a, b); }
#define RG_PG(A, DP, VEC) { if (whole) RG_PG_(A, DP, VEC, true) RG_PG_(A, DP, VEC, false) }
#define RG_PG_WIDTH(A, VEC) { if (a.d <= 32) RG_PG(A, 32, VEC) if (a.d <= 64) RG_PG(A, 64, VEC) RG_PG(A, 128, VEC) }
    if (dtype == RG_DTYPE_F32) { if (vec) RG_PG_WIDTH(float, true) RG_PG_WIDTH(float, false) }
    if (vec) RG_PG_WIDTH(bf16, true)
    RG_PG_WIDTH(bf16, false)
#undef RG_PG_WIDTH
#undef RG_PG
#undef RG_PG_
}

// bfloat16, head sizes in pieces of 64, pages of a power of two from 8 on, rows on 4-byte boundaries, and addresses that fit
// the map's coordinates.
static bool parts_mma_ok(const PartArgs& a, int dtype, int num_pages) {
    return dtype == RG_DTYPE_BF16 && a.d % 64 == 0 && a.page_shift >= 3 && a.q_stride % 2 == 0 && ((uintptr_t)a.q & 3) == 0 &&
           ((uintptr_t)a.kv & 15) == 0 && (long long)num_pages * 2 * a.nkv * a.page_size < 0x7fffffffll && a.score_ld % 2 == 0;
}

static int launch_parts_mma(const PartArgs& a, int num_pages, int* err, cudaStream_t s) {
    const long long blocks = part_blocks(a);
    if (blocks > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
    if (blocks == 0) return 0;
    CUtensorMap map;
    int e = make_kv_map(&map, a.kv, num_pages, a.nkv, a.page_size, a.d, a.page_size < 16 ? a.page_size : 16);
    if (e) return e;
#define RG_PM(P, B) { constexpr int smem = 4 * pm_stages(P, B) * pm_stage_bytes(P) + 1024; \
    RG_ALLOW_SMEM((parts_mma_kernel<P, B>), smem) \
    return rg_launch(parts_mma_kernel<P, B>, dim3((unsigned)blocks), dim3(PM_THREADS), smem, s, 1, map, a, err); }
    const bool brief = pm_brief(a.d, max(a.n_groups ? a.prefix_per : 0, a.own_per), blocks);
    if (a.d == 64) { if (brief) RG_PM(1, true) else RG_PM(1, false) }
    if (a.d == 128) { if (brief) RG_PM(2, true) else RG_PM(2, false) }
    if (a.d == 192) RG_PM(3, false)
    RG_PM(4, false)
#undef RG_PM
}

// Rows by clusters of `cluster` blocks, in one launch; b.weights null: no weights.
static int launch_rows(const PartArgs& a, const RowsArgs& b, int dtype, int num_pages, int cluster, int* err, cudaStream_t s) {
    if (cluster > 8) return RG_ERR_UNSUPPORTED;
    if (!parts_mma_ok(a, dtype, num_pages)) return launch_parts_general(a, dtype, s, &b, cluster);
    if (a.nkv * a.own_tiles > 65535 || (long long)cluster * a.T > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
    CUtensorMap map;
    int e = make_kv_map(&map, a.kv, num_pages, a.nkv, a.page_size, a.d, a.page_size < 16 ? a.page_size : 16);
    if (e) return e;
    const int scores = b.weights ? (a.nh / a.nkv) * (b.runs * 16 + 8) * 4 : 0;
    const dim3 grid(cluster * a.T, a.nkv * a.own_tiles);
#define RG_RM(P, W, B) { constexpr int stages = 4 * pm_stages(P, B) * pm_stage_bytes(P) + 1024; \
    RG_ALLOW_SMEM((rows_mma_kernel<P, W, B>), 227 * 1024 - 2048) \
    return rg_launch(rows_mma_kernel<P, W, B>, grid, dim3(PM_THREADS), stages + scores, s, cluster, map, a, b, err); }
#define RG_RMW(P, B) { if (b.weights) RG_RM(P, true, B) else RG_RM(P, false, B) }
    const bool brief = pm_brief(a.d, ((long long)a.prefix_limit + a.own_limit + cluster - 1) / cluster, (long long)grid.x * grid.y);
    if (a.d == 64) { if (brief) RG_RMW(1, true) else RG_RMW(1, false) }
    if (a.d == 128) { if (brief) RG_RMW(2, true) else RG_RMW(2, false) }
    if (a.d == 192) RG_RMW(3, false)
    RG_RMW(4, false)
#undef RG_RMW
#undef RG_RM
}

static int launch_parts(const PartArgs& a, int dtype, int num_pages, int* err, cudaStream_t s) {
    return parts_mma_ok(a, dtype, num_pages) ? launch_parts_mma(a, num_pages, err, s) : launch_parts_general(a, dtype, s);
}

static bool fill_part_args(PartArgs& a, const void* q, int q_stride, const void* kv, const int* block_table, int max_blocks,
                           const int* positions, int T, int nh, int nkv, int d, int page_size, float scale, float* part_o,
                           float* part_ml, int own_parts, int own_per) {
    if (T < 0 || d < 1 || d > 256 || nkv < 1 || nh < nkv || nh % nkv || page_size < 1 || own_parts < 0 || own_per < 1 ||
        ((uintptr_t)part_o & 15) || ((uintptr_t)part_ml & 7))        // outputs are read in fours, (m, l) in pairs
        return false;
    a = PartArgs{};
    a.q = q; a.q_stride = q_stride; a.kv = kv; a.block_table = block_table; a.max_blocks = max_blocks; a.positions = positions;
    a.T = T; a.nh = nh; a.nkv = nkv; a.d = d; a.page_size = page_size; a.scale_log2 = scale * 1.4426950408889634f;
    a.part_o = part_o; a.part_ml = part_ml; a.own_parts = own_parts; a.own_per = own_per; a.prefix_per = 1;
    a.page_shift = -1;
    for (int b = 0; b < 31; ++b) if (page_size == (1 << b)) a.page_shift = b;
    const long long room = (long long)max_blocks * page_size, cut = (long long)own_parts * own_per;
    a.own_limit = (int)min(0x7fffffffll, min(room, cut));
    return true;
}

// Rows of single tokens behind shared prefixes: see attention_parts.cuh for the arguments.  Scratch: part_o
// [T, nh, prefix_parts + own_parts, d] on a 16-byte boundary and part_ml [.., 2] on one of 8.  tensor_cores: 1 the prefixes by
// prefix_tc_kernel, 2 the same with two parts a block (groups of up to 128 queries a kv head), 0 everything in one launch.  cluster:
// not 0, rows by clusters of so many blocks, which leave no parts.  max_prefix, max_own: the most entries of either list that are seen.
extern "C" int rg_prefix_attention(const void* q, int q_stride, void* out, int out_ld, const void* kv, int num_pages, int dtype,
                                   const int* prefix_table, int prefix_blocks, const int* groups, int n_groups, int max_rows,
                                   int prefix_parts, int prefix_per, const int* block_table, int max_blocks, const int* positions,
                                   int own_parts, int own_per, int T, int nh, int nkv, int d, int page_size, float scale,
                                   float* part_o, float* part_ml, int max_prefix, int max_own, int tensor_cores, int cluster,
                                   int* err, void* stream) {
    if (T <= 0) return 0;
    PartArgs a;
    if (!fill_part_args(a, q, q_stride, kv, block_table, max_blocks, positions, T, nh, nkv, d, page_size, scale, part_o, part_ml,
                        own_parts, own_per) || n_groups < 0 || prefix_parts < 0 || prefix_per < 1 || out_ld < nh * d || max_prefix < 0 ||
        max_own < 0)
        return RG_ERR_UNSUPPORTED;
    const int group = nh / nkv;
    a.prefix_table = prefix_table; a.prefix_blocks = prefix_blocks; a.groups = groups; a.n_groups = n_groups; a.max_rows = max_rows;
    a.prefix_parts = prefix_parts; a.prefix_per = prefix_per;
    // parts are whole tiles: where they end is behind what the call says may be seen
    a.prefix_limit = (int)min((long long)max_prefix, min((long long)prefix_blocks * page_size, (long long)prefix_parts * prefix_per));
    a.own_limit = min(a.own_limit, max_own);
    if ((long long)max_rows * group > 0x7fffff00ll || (long long)T * nh > 0x7fffffffll) return RG_ERR_UNSUPPORTED;   // rounded up to tiles below
    a.own_tiles = (group + PG_Q - 1) / PG_Q;
    if (cluster) {
        const RowsArgs b = {out, nullptr, nullptr, 0, out_ld, 0, 0, 0.f};
        return launch_rows(a, b, dtype, num_pages, cluster, err, (cudaStream_t)stream);
    }
    if (tensor_cores) {
        if (!prefix_tc_ok(a, dtype, num_pages)) return RG_ERR_UNSUPPORTED;
        const int tile_rows = (tensor_cores == 2 ? 1 : 2) * (PT_SIDE / group);
        a.prefix_tiles = (max_rows + tile_rows - 1) / tile_rows;
        int e = launch_prefix_tc(a, num_pages, tensor_cores == 2, err, (cudaStream_t)stream);
        if (e) return e;
        PartArgs own = a;                                            // their own entries, beside the prefixes
        own.n_groups = 0;
        own.beside = a.n_groups > 0 && rg_pdl_enabled;
        e = launch_parts(own, dtype, num_pages, err, (cudaStream_t)stream);
        if (e) return e;
    } else {
        a.prefix_tiles = (max_rows * group + PG_Q - 1) / PG_Q;
        int e = launch_parts(a, dtype, num_pages, err, (cudaStream_t)stream);
        if (e) return e;
    }
    if (dtype == RG_DTYPE_F32)
        return rg_launch(join_kernel<float>, dim3(join_blocks(a)), dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a, join_heads(a), (float*)out, out_ld);
    return rg_launch(join_kernel<bf16>, dim3(join_blocks(a)), dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a, join_heads(a), (bf16*)out, out_ld);
}

// Single tokens with the weights of their entries.  weights [n_slots, nkv, weights_ld]; scores [T, nh, score_ld] is scratch.
extern "C" int rg_weighed_attention(const void* q, int q_stride, void* out, int out_ld, const void* kv, int num_pages, int dtype,
                                    const int* block_table, int max_blocks, const int* positions, int own_parts, int own_per,
                                    int T, int nh, int nkv, int d, int page_size, float scale, float* part_o, float* part_ml,
                                    float* scores, int score_ld, float* weights, int weights_ld, int n_slots, const int* slots,
                                    int max_context, float decay, int cluster, int* err, void* stream) {
    if (T <= 0) return 0;
    PartArgs a;
    if (!fill_part_args(a, q, q_stride, kv, block_table, max_blocks, positions, T, nh, nkv, d, page_size, scale, part_o, part_ml,
                        own_parts, own_per) || max_context > score_ld || max_context > weights_ld || out_ld < nh * d)
        return RG_ERR_UNSUPPORTED;
    if (score_ld % 4 || ((uintptr_t)scores & 15)) return RG_ERR_UNSUPPORTED;   // read in fours
    a.scores = scores; a.score_ld = score_ld;
    a.own_limit = min(a.own_limit, max_context);
    const int group = nh / nkv;
    a.own_tiles = (group + PG_Q - 1) / PG_Q;
    if (cluster) {                                                   // own_per: the most entries a block may have
        if (a.own_tiles != 1 || own_per % 16) return RG_ERR_UNSUPPORTED;
        const RowsArgs b = {out, weights, slots, weights_ld, out_ld, n_slots, own_per / 16, decay};
        return launch_rows(a, b, dtype, num_pages, cluster, err, (cudaStream_t)stream);
    }
    int e = launch_parts(a, dtype, num_pages, err, (cudaStream_t)stream);
    if (e) return e;
    const int chunks = (max_context + WEIGH_CHUNK - 1) / WEIGH_CHUNK;
    const long long blocks = join_blocks(a) + (long long)T * nkv * chunks;
    if (blocks > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
    if (dtype == RG_DTYPE_F32)
        return rg_launch(weigh_kernel<float>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a,
                         (int)join_blocks(a), join_heads(a), (float*)out, out_ld, weights, (long long)weights_ld, n_slots, slots, chunks, decay);
    return rg_launch(weigh_kernel<bf16>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a,
                     (int)join_blocks(a), join_heads(a), (bf16*)out, out_ld, weights, (long long)weights_ld, n_slots, slots, chunks, decay);
}
