// Attention of trees of drafted tokens over the paged cache and over one another.  attention_tree.cuh says what is computed and
// how it is cut.
#include "attention_tree.cuh"
#include "attention_tree_tcgen05.cuh"
#include "mma.cuh"

#define TG_THREADS 128
#define TG_Q 16                // queries of an item
#define TG_K 64                // entries of a tile
#define TG_LD (TG_K + 4)

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

__host__ __device__ inline int tg_row(int d) { return ((d + 3) & ~3) + 4; }   // floats a row in shared memory
__host__ __device__ inline int tg_stages(int d) { return d <= 128 ? 2 : 1; }   // tiles of K and V in shared memory: the next one is on its way

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

// ---------------------------------------------------------------------------------------------------
// Any head size up to 256, any page size, 32-bit or bfloat16 storage, all arithmetic in 32-bit.
// Per tile of 64 entries: 2 queries x 4 entries of scores a thread, then a column of the output for all 16 queries a thread;
// DP = 32 or 64: as many threads share the columns, and TG_THREADS / DP groups of them share the tile's entries.
// ---------------------------------------------------------------------------------------------------
template <typename A, int DP, bool VEC>
__global__ void __launch_bounds__(TG_THREADS) tree_general_kernel(const TreeArgs a) {
    extern __shared__ __align__(16) float smem[];
    constexpr int GROUPS = TG_THREADS / DP, COLS = DP == 128 ? 2 : 1;
    __shared__ TreeStart st;
    __shared__ long long row_at[2][TG_K];                           // where the rows of a tile are in the cache, -1 behind its end
    pdl_wait();
    pdl_trigger();
    tree_plan<TG_THREADS>(a, blockIdx.x, 1, 0, st);
    if (st.r[0] < 0) return;
    const int d = a.d, ld = tg_row(d), group = a.nh / a.nkv, tid = threadIdx.x, stages = tg_stages(d);
    float* qs = smem;                                               // [16][ld]
    float* kv0 = qs + TG_Q * ld;                                    // [stages][K [64][ld], V [64][ld]]
    float* ps = kv0 + stages * 2 * TG_K * ld;                       // [16][TG_LD]
    float* al = ps + TG_Q * TG_LD;                                  // [16]
    const size_t to_values = (size_t)a.nkv * a.page_size * d;
    const int n_tiles = (int)min(st.per, st.total - (long long)blockIdx.x * st.per);
    TreeWalk w, ahead;                                              // this tile, and the one whose rows are looked up
    w.at(a, st.r[0], st.in[0]);
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
    int q0 = 0, nq = 0;
    look_up(0);
    look_up(1);
    __syncthreads();
    if (stages == 2) request(0, kv0);
    for (int step = 0; step < n_tiles; ++step) {
        if (step == 0 || w.tile == 0) {                                // an item begins
            q0 = w.block() * TG_Q;
            nq = min(TG_Q, w.x.rows * group - q0);
            for (int j = tid; j < TG_Q * ld; j += TG_THREADS) {     // nobody reads the last item's any more
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
        }
        const int slot = step & 1, e0 = w.tile * TG_K, n = min(TG_K, w.x.entries - e0);
        float* ks = kv0 + (stages == 2 ? slot * 2 * TG_K * ld : 0);
        const float* vs = ks + TG_K * ld;
        if (stages == 1) {
            __syncthreads();                                        // the last tile's values are read
            request(slot, ks);
        }
        rgmma::cp_async_wait<0>();
        __syncthreads();                                            // the tile is there; with two stages the last one is read
        if (stages == 2 && step + 1 < n_tiles) request(slot ^ 1, kv0 + (slot ^ 1) * 2 * TG_K * ld);
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
        if (step + 1 == n_tiles || w.last_tile()) {                    // the item, or the stretch, ends: leave the part
            float sums[2] = {l[0], l[1]};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], o);
            }
            const size_t place = (size_t)w.first_query(a) + (size_t)blockIdx.x * TG_Q;
            if constexpr (GROUPS > 1) {                             // the groups' sums, added in their order, through this tile's K and V
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
                        a.part_ml[(place + 2 * qa + i) * 2] = m[i];
                        a.part_ml[(place + 2 * qa + i) * 2 + 1] = sums[i];
                    }
            __syncthreads();                                        // the queries, and what went through the tile, are read
        }
        w.next(a, step + 1 < n_tiles);
    }
}

// ---------------------------------------------------------------------------------------------------
// Joining the parts of a row and head.
// ---------------------------------------------------------------------------------------------------
#define JOIN_THREADS 128

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
// sum.  For rows whose output is no number or infinite: 0, the weight of an entry that is not seen, times such a value is no number.
template <typename A>
__device__ __noinline__ void row_by_formula(const TreeArgs& a, const TreeRequest& x, int r, int t, int h, A* to) {
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
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (lane + 32 * k < d) to[lane + 32 * k] = from_f32<A>(acc[k] * inv);
}

// One warp joins row t and head h, parts in their order; 4 columns a lane.
template <typename A>
__global__ void __launch_bounds__(JOIN_THREADS) tree_join_kernel(const TreeArgs a, A* __restrict__ out, int out_ld) {
    pdl_wait();
    pdl_trigger();
    const long long i = (long long)blockIdx.x * (JOIN_THREADS / 32) + (threadIdx.x >> 5);
    const int t = (int)(i / a.nh), h = (int)(i % a.nh), lane = threadIdx.x & 31;
    if (t >= a.T) return;
    const int r = request_of(a, t);
    if (r < 0) return;
    const TreeRequest x = tree_request(a, r);
    if (t - x.row0 >= x.rows) return;                               // more rows than the call says
    const int d = a.d, group = a.nh / a.nkv, kvh = h / group, qi = (t - x.row0) * group + h % group, block = qi / a.item_queries;
    const long long per = a.plan[a.R], tile0 = a.plan[r] + ((long long)kvh * x.blocks + block) * x.tiles;
    const int w0 = (int)(tile0 / per), n = x.tiles ? (int)((tile0 + x.tiles - 1) / per) - w0 + 1 : 0;
    // the row's place in the first part; the next part's is item_queries further
    const size_t place = (size_t)x.row0 * a.nh + (size_t)kvh * x.rows * group + qi + (size_t)w0 * a.item_queries;
    float M = -INFINITY, L = 0.f;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, a.part_ml[(place + (size_t)i * a.item_queries) * 2]);
    M = warp_max(M);
    if (M == -INFINITY) M = 0.f;
    for (int i = lane; i < n; i += 32) {
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + (place + (size_t)i * a.item_queries) * 2);
        L += ml.y * exp2f(ml.x - M);
    }
    L = warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    A* to = out + (size_t)t * out_ld + (size_t)h * d;
    bool odd = false;
    for (int c0 = 0; c0 < d; c0 += 128) {
        const int c = c0 + 4 * lane;
        float4 acc = {0.f, 0.f, 0.f, 0.f};
        for (int i0 = 0; i0 < n; i0 += 32) {
            float f = 0.f;
            if (i0 + lane < n) f = exp2f(a.part_ml[(place + (size_t)(i0 + lane) * a.item_queries) * 2] - M) * inv;
            const int some = min(32, n - i0);
#pragma unroll 4
            for (int i = 0; i < some; ++i) {
                const float fi = __shfl_sync(0xffffffffu, f, i);
                const float* from = a.part_o + (place + (size_t)(i0 + i) * a.item_queries) * d + c;
                float4 y = {0.f, 0.f, 0.f, 0.f};
                if (d % 4 == 0) { if (c < d) y = *reinterpret_cast<const float4*>(from); }
                else { if (c < d) y.x = from[0]; if (c + 1 < d) y.y = from[1]; if (c + 2 < d) y.z = from[2]; if (c + 3 < d) y.w = from[3]; }
                acc.x += fi * y.x; acc.y += fi * y.y; acc.z += fi * y.z; acc.w += fi * y.w;
            }
        }
        odd |= !(isfinite(acc.x) && isfinite(acc.y) && isfinite(acc.z) && isfinite(acc.w));
        if (c < d) to[c] = from_f32<A>(acc.x);
        if (c + 1 < d) to[c + 1] = from_f32<A>(acc.y);
        if (c + 2 < d) to[c + 2] = from_f32<A>(acc.z);
        if (c + 3 < d) to[c + 3] = from_f32<A>(acc.w);
    }
    if (__any_sync(0xffffffffu, odd)) row_by_formula<A>(a, x, r, t, h, to);
}

// ---------------------------------------------------------------------------------------------------
static size_t tg_smem(int d) { return (size_t)((TG_Q + tg_stages(d) * 2 * TG_K) * tg_row(d) + TG_Q * TG_LD + TG_Q) * sizeof(float); }

static int launch_tree_general(const TreeArgs& a, int dtype, cudaStream_t s) {
    const size_t smem = tg_smem(a.d);
    const bool vec = a.d % 4 == 0 && (((uintptr_t)a.kv) & (dtype == RG_DTYPE_F32 ? 15 : 7)) == 0;
#define RG_TG(A, DP, VEC) { RG_ALLOW_SMEM((tree_general_kernel<A, DP, VEC>), 160 * 1024) \
    return rg_launch(tree_general_kernel<A, DP, VEC>, dim3((unsigned)a.workers), dim3(TG_THREADS), smem, s, 1, a); }
#define RG_TG_WIDTH(A, VEC) { if (a.d <= 32) RG_TG(A, 32, VEC) if (a.d <= 64) RG_TG(A, 64, VEC) RG_TG(A, 128, VEC) }
    if (dtype == RG_DTYPE_F32) { if (vec) RG_TG_WIDTH(float, true) RG_TG_WIDTH(float, false) }
    if (vec) RG_TG_WIDTH(bf16, true)
    RG_TG_WIDTH(bf16, false)
#undef RG_TG_WIDTH
#undef RG_TG
}

// See attention_tree.cuh for the arguments.  Scratch: plan [R + 1] on an 8-byte boundary, part_o [T nh + workers item_queries, d]
// on one of 32 bytes and part_ml [.., 2] on one of 8.  tensor_cores: 0 tree_general_kernel; 1 tree_tc_kernel, a stretch a side; 2 the same,
// a stretch for both sides; tile_rows: rows of a side.
extern "C" int rg_tree_attention(const void* q, int q_stride, void* out, int out_ld, const void* kv, int num_pages, int dtype,
                                 const int* block_table, int max_blocks, const int* cu_rows, const int* starts, const int* masks, int words,
                                 int R, int T, int nh, int nkv, int d, int page_size, float scale, int max_rows, int max_context,
                                 int blocks, int workers, int item_queries, int least, int tile_rows, int tensor_cores, float* part_o, float* part_ml, long long* plan, int* err, void* stream) {
    if (T <= 0 || R <= 0 || max_rows <= 0) return 0;
    if (d < 1 || d > 256 || nkv < 1 || nh < nkv || nh % nkv || page_size < 1 || max_blocks < 0 || words < 0 || max_context < 0 || out_ld < nh * d ||
        workers < 1 || item_queries < 1 || least < 1 || ((uintptr_t)part_o & 31) || ((uintptr_t)part_ml & 7) || ((uintptr_t)plan & 7) ||
        (long long)T * nh > 0x7fffffffll)
        return RG_ERR_UNSUPPORTED;
    TreeArgs a = {};
    a.q = q; a.q_stride = q_stride; a.kv = kv; a.block_table = block_table; a.max_blocks = max_blocks; a.cu_rows = cu_rows; a.starts = starts;
    a.masks = masks; a.words = words; a.R = R; a.T = T; a.nh = nh; a.nkv = nkv; a.d = d; a.page_size = page_size; a.pages = num_pages;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.max_rows = max_rows;
    a.limit = (int)min((long long)max_context, min(0x7fffff00ll, (long long)max_blocks * page_size));
    a.workers = workers; a.item_queries = item_queries; a.least = least;
    a.part_o = part_o; a.part_ml = part_ml; a.plan = plan; a.err = err;
    a.page_shift = -1;
    for (int b = 0; b < 31; ++b) if (page_size == (1 << b)) a.page_shift = b;
    a.tile = tensor_cores ? TT_STAGE : TG_K;
    if (tensor_cores ? !tree_tc_ok(a, dtype) : item_queries != TG_Q || workers != blocks) return RG_ERR_UNSUPPORTED;
    int e = tensor_cores ? launch_tree_tc(a, tile_rows, tensor_cores == 2, blocks, (cudaStream_t)stream) : launch_tree_general(a, dtype, (cudaStream_t)stream);
    if (e) return e;
    const long long joins = ((long long)T * nh + JOIN_THREADS / 32 - 1) / (JOIN_THREADS / 32);
    if (dtype == RG_DTYPE_F32)
        return rg_launch(tree_join_kernel<float>, dim3((unsigned)joins), dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a, (float*)out, out_ld);
    return rg_launch(tree_join_kernel<bf16>, dim3((unsigned)joins), dim3(JOIN_THREADS), 0, (cudaStream_t)stream, 1, a, (bf16*)out, out_ld);
}
