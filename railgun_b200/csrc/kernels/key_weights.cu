// The weights that cached entries receive from portions of prompts:
//   w[e] (+)= sum over the portion's rows t at positions p_t >= e and the heads h of a kv head of 2^(s_th(e) - z_th),
//   s = scale log2(e) q.k,   z_th = log2 sum_e 2^(s_th(e))
// in two passes over the scores: z first, then the sums.  A block of the second pass owns its entries and goes over all
// rows that see them, so sums have one order and need no atomics.
#include "common.cuh"

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
};

// Request r's rows and entries, cut to what there is room for.
__device__ __forceinline__ void rows_of(const WeightArgs& a, int r, int& row0, int& rows, int& start, int& entries) {
    row0 = max(0, a.cu_rows[r]);
    rows = min(a.cu_rows[r + 1], a.T) - row0;
    start = a.starts[r];
    entries = rows > 0 && start >= 0 ? min(start + rows, a.limit) : 0;
}

// ---------------------------------------------------------------------------------------------------
// Any head size up to 256, any page size, 32-bit or bfloat16 storage, all arithmetic in 32-bit.  16 queries (rows x heads
// of a kv head) by 64 entries at a time, 2 x 4 a thread.
// ---------------------------------------------------------------------------------------------------
#define KW_THREADS 128
#define KW_Q 16
#define KW_K 64

template <typename A>
__device__ __forceinline__ void load_queries(const WeightArgs& a, float* qs, int ld, int row0, int kvh, int q0, int nq) {
    const int group = a.nh / a.nkv;
    for (int i = threadIdx.x; i < KW_Q * ld; i += KW_THREADS) {
        const int row = i / ld, c = i - row * ld, qi = q0 + row;
        float v = 0.f;
        if (row < nq && c < a.d)
            v = to_f32(((const A*)a.q)[(size_t)(row0 + qi / group) * a.q_stride + (kvh * group + qi % group) * a.d + c]) * a.scale_log2;
        qs[i] = v;
    }
}
template <typename A>
__device__ __forceinline__ void load_keys(const WeightArgs& a, float* ks, int ld, const int* table, int kvh, int e0, int n) {
    const size_t page_elems = (size_t)2 * a.nkv * a.page_size * a.d;
    for (int i = threadIdx.x; i < KW_K * ld; i += KW_THREADS) {
        const int row = i / ld, c = i - row * ld, e = e0 + row;
        float v = 0.f;
        if (row < n && c < a.d)
            v = to_f32(((const A*)a.kv)[(size_t)table[e / a.page_size] * page_elems + ((size_t)kvh * a.page_size + e % a.page_size) * a.d + c]);
        ks[i] = v;
    }
}
__device__ __forceinline__ void tile_scores(float (&sc)[2][4], const float* qs, const float* ks, int ld, int d, int qa, int ka) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
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
}

__host__ __device__ inline int kw_row(int d) { return ((d + 3) & ~3) + 4; }

// grid (query tiles, nkv, R)
template <typename A>
__global__ void __launch_bounds__(KW_THREADS) row_sums_general_kernel(const WeightArgs a) {
    extern __shared__ __align__(16) float smem[];
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y, group = a.nh / a.nkv, q0 = blockIdx.x * KW_Q;
    int row0, rows, start, entries;
    rows_of(a, r, row0, rows, start, entries);
    const int nq = min(KW_Q, rows * group - q0);
    if (nq <= 0 || entries <= 0) return;
    const int ld = kw_row(a.d), qa = threadIdx.x >> 4, ka = threadIdx.x & 15;
    float *qs = smem, *ks = smem + KW_Q * ld;
    load_queries<A>(a, qs, ld, row0, kvh, q0, nq);
    const int* table = a.block_table + (size_t)r * a.max_blocks;
    const int last = min(entries, start + (q0 + nq - 1) / group + 1);          // what the tile's last row sees
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int e0 = 0; e0 < last; e0 += KW_K) {
        const int n = min(KW_K, last - e0);
        __syncthreads();
        load_keys<A>(a, ks, ld, table, kvh, e0, n);
        __syncthreads();
        float sc[2][4];
        tile_scores(sc, qs, ks, ld, a.d, qa, ka);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int sees = min(n, start + (q0 + 2 * qa + i) / group + 1 - e0);
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
    for (int i = 0; i < 2; ++i) {
        float M = m[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float ms = M == -INFINITY ? 0.f : M;
        float L = l[i] * exp2f(m[i] - ms);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        const int qi = q0 + 2 * qa + i;
        if (ka == 0 && 2 * qa + i < nq)                             // no weight at all: every 2^(s - z) is 0
            a.z[(size_t)(row0 + qi / group) * a.nh + kvh * group + qi % group] = L > 0.f ? ms + log2f(L) : INFINITY;
    }
}

// grid (tiles of entries, nkv, R)
template <typename A>
__global__ void __launch_bounds__(KW_THREADS) entry_sums_general_kernel(const WeightArgs a) {
    extern __shared__ __align__(16) float smem[];
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.z, kvh = blockIdx.y, group = a.nh / a.nkv, e0 = blockIdx.x * KW_K, slot = a.slots[r];
    int row0, rows, start, entries;
    rows_of(a, r, row0, rows, start, entries);
    const int n = min(KW_K, entries - e0);
    if (n <= 0 || slot < 0 || slot >= a.n_slots) return;
    const int ld = kw_row(a.d), qa = threadIdx.x >> 4, ka = threadIdx.x & 15;
    float *qs = smem, *ks = qs + KW_Q * ld, *part = ks + KW_K * ld;            // part [8][64]
    load_keys<A>(a, ks, ld, a.block_table + (size_t)r * a.max_blocks, kvh, e0, n);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int q0 = max(0, e0 - start) * group; q0 < rows * group; q0 += KW_Q) {  // from the first row that sees entry e0
        const int nq = min(KW_Q, rows * group - q0);
        __syncthreads();
        load_queries<A>(a, qs, ld, row0, kvh, q0, nq);
        __syncthreads();
        float sc[2][4];
        tile_scores(sc, qs, ks, ld, a.d, qa, ka);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (2 * qa + i >= nq) continue;
            const int qi = q0 + 2 * qa + i, sees = start + qi / group + 1 - e0;
            const float z = a.z[(size_t)(row0 + qi / group) * a.nh + kvh * group + qi % group];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (ka + 16 * j < sees) sum[j] += exp2f(sc[i][j] - z);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) part[qa * KW_K + ka + 16 * j] = sum[j];
    __syncthreads();
    float* w = a.weights + ((size_t)slot * a.nkv + kvh) * a.weights_ld + e0;
    if (threadIdx.x < n) {
        float v = e0 + (int)threadIdx.x < a.fresh[r] ? w[threadIdx.x] : 0.f;
        float added = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) added += part[i * KW_K + threadIdx.x];
        w[threadIdx.x] = v + added;
    }
}

// z [T, nh] is scratch; max_rows: the most rows of a request; max_context: the most entries a row sees.
extern "C" int rg_prompt_key_weights(const void* q, int q_stride, const void* kv, int dtype, float* weights, int weights_ld,
                                     int n_slots, const int* slots, const int* block_table, int max_blocks, const int* cu_rows,
                                     const int* starts, const int* fresh, int R, int T, int nh, int nkv, int d, int page_size,
                                     float scale, int max_rows, int max_context, float* z, void* stream) {
    if (R <= 0 || T <= 0 || max_rows <= 0 || max_context <= 0) return 0;
    if (d < 1 || d > 256 || nkv < 1 || nh < nkv || nh % nkv || page_size < 1 || max_context > weights_ld || R > 65535 || nkv > 65535 ||
        (long long)max_rows * (nh / nkv) > 0x7fffffffll)
        return RG_ERR_UNSUPPORTED;
    const WeightArgs a = {q, kv, block_table, cu_rows, starts, fresh, slots, weights, z, weights_ld, q_stride, max_blocks, n_slots, T, R,
                          nh, nkv, d, page_size, (int)min((long long)max_context, (long long)max_blocks * page_size),
                          scale * 1.4426950408889634f};
    const cudaStream_t s = (cudaStream_t)stream;
    const size_t smem = (size_t)((KW_Q + KW_K) * kw_row(d) + 8 * KW_K) * sizeof(float);
    const dim3 by_query((max_rows * (nh / nkv) + KW_Q - 1) / KW_Q, nkv, R), by_entry((max_context + KW_K - 1) / KW_K, nkv, R);
#define RG_KW(A) { cudaError_t ce = cudaFuncSetAttribute(row_sums_general_kernel<A>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); \
    if (ce == cudaSuccess) ce = cudaFuncSetAttribute(entry_sums_general_kernel<A>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); \
    if (ce != cudaSuccess) return (int)ce; \
    const int e = rg_launch(row_sums_general_kernel<A>, by_query, dim3(KW_THREADS), smem, s, 1, a); \
    return e ? e : rg_launch(entry_sums_general_kernel<A>, by_entry, dim3(KW_THREADS), smem, s, 1, a); }
    if (dtype == RG_DTYPE_F32) RG_KW(float)
    RG_KW(bf16)
#undef RG_KW
}
