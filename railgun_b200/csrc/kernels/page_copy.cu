// Copies of pages in several caches at once.
//
// A cache is [pages, outer, page, inner bytes]: of a copy (from, to, held) the first `held` of the page's entries are copied, which
// are one run of held x inner bytes for each of `outer`.  Nothing but the bytes themselves goes to memory or comes from it: where the
// caches are, and the copies, are arguments of the kernel.  256 pages of 28 layers (24 heads on 8 of 128, 499 MB there and back) take
// 77 us, 98 % of what a plain copy reaches; 8 pages of 9 entries in 16 layers 2.1, the launch and a trip each way.
#include "common.cuh"
#include <cstdlib>

#define COPY_THREADS 256
#define COPY_AHEAD 8                   // loads that a lane has under way
#define COPY_CACHES 64
#define COPY_MOST 256                  // of a launch
#define RG_COPY_RANGE 10002            // a page or a number of entries that the caches do not have
#define RG_COPY_TWICE 10003            // a page that is written twice, or written and read

struct CopyArgs {
    char* at[COPY_CACHES];
    int from[COPY_MOST], to[COPY_MOST], held[COPY_MOST];
    long long page_bytes, run_bytes;   // of a page, and of a run of a whole page's entries
    int n_caches, n, outer, inner;     // inner: bytes of an entry
    int pieces;                        // a warp's pieces of a whole run
};

// A warp takes pieces of 32 x COPY_AHEAD units of a run.
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const long long all = (long long)a.n_caches * a.n * a.outer * a.pieces;
    for (long long i = (long long)blockIdx.x * (COPY_THREADS / 32) + (threadIdx.x >> 5); i < all; i += (long long)gridDim.x * (COPY_THREADS / 32)) {
        const int piece = (int)(i % a.pieces);
        long long rest = i / a.pieces;
        const int o = (int)(rest % a.outer);
        rest /= a.outer;
        const int k = (int)(rest % a.n), cache = (int)(rest / a.n);
        const long long units = (long long)a.held[k] * a.inner / (long long)sizeof(V), u0 = (long long)piece * (32 * COPY_AHEAD) + lane;
        const V* from = reinterpret_cast<const V*>(a.at[cache] + a.from[k] * a.page_bytes + o * a.run_bytes);
        V* to = reinterpret_cast<V*>(a.at[cache] + a.to[k] * a.page_bytes + o * a.run_bytes);
        V v[COPY_AHEAD];
#pragma unroll
        for (int j = 0; j < COPY_AHEAD; ++j)
            if (u0 + 32 * j < units) v[j] = from[u0 + 32 * j];
#pragma unroll
        for (int j = 0; j < COPY_AHEAD; ++j)
            if (u0 + 32 * j < units) to[u0 + 32 * j] = v[j];
    }
}

// copies [n][3] on the host: from, to, entries held (-1: all).  unit: bytes (1, 2, 4, 8 or 16) that entries and addresses are multiples of.
extern "C" int rg_copy_pages(const unsigned long long* caches, int n_caches, int pages, int outer, int page_size, long long inner_bytes, int unit,
                             const int* copies, int n, int sms, void* stream) {
    if (n <= 0) return 0;
    if (n_caches < 1 || pages < 0 || outer < 1 || page_size < 1 || inner_bytes < 1 || inner_bytes > 0x7fffffffll || unit < 1 ||
        inner_bytes % unit || sms < 1)
        return RG_ERR_UNSUPPORTED;
    unsigned char* used = (unsigned char*)calloc((size_t)pages + 1, 1);       // 1: written, 2: read
    if (!used) return (int)cudaErrorMemoryAllocation;
    int bad = 0;
    for (int i = 0; i < n && !bad; ++i) {
        const int from = copies[3 * i], to = copies[3 * i + 1], held = copies[3 * i + 2];
        if (from < 0 || from >= pages || to < 0 || to >= pages || held < -1 || held > page_size) bad = RG_COPY_RANGE;
        else if (from != to && used[to]) bad = RG_COPY_TWICE;
        else if (from != to && (used[from] & 1)) bad = RG_COPY_TWICE;
        else if (from != to) { used[to] |= 1; used[from] |= 2; }
    }
    free(used);
    if (bad) return bad;
    for (int c0 = 0; c0 < n_caches; c0 += COPY_CACHES)
        for (int k0 = 0; k0 < n;) {
            CopyArgs a = {};
            a.n_caches = n_caches - c0 < COPY_CACHES ? n_caches - c0 : COPY_CACHES;
            for (int i = 0; i < a.n_caches; ++i) {
                if (caches[c0 + i] % unit) return RG_ERR_UNSUPPORTED;
                a.at[i] = reinterpret_cast<char*>(caches[c0 + i]);
            }
            for (; k0 < n && a.n < COPY_MOST; ++k0) {
                const int* c = copies + 3 * k0;
                const int held = c[2] < 0 ? page_size : c[2];
                if (c[0] == c[1] || held == 0) continue;
                a.from[a.n] = c[0]; a.to[a.n] = c[1]; a.held[a.n] = held;
                ++a.n;
            }
            if (a.n == 0) continue;
            a.outer = outer; a.inner = (int)inner_bytes;
            a.run_bytes = page_size * inner_bytes;
            a.page_bytes = outer * a.run_bytes;
            const long long piece_bytes = 32ll * COPY_AHEAD * unit, pieces = (a.run_bytes + piece_bytes - 1) / piece_bytes;
            if (pieces > 0x7fffffffll) return RG_ERR_UNSUPPORTED;
            a.pieces = (int)pieces;
            const long long warps = (long long)a.n_caches * a.n * outer * pieces, blocks = (warps + COPY_THREADS / 32 - 1) / (COPY_THREADS / 32),
                            most = 8ll * sms;
            const dim3 grid((unsigned)(blocks < most ? blocks : most));
            int e;
            switch (unit) {
                case 16: e = rg_launch(copy_pages_kernel<uint4>, grid, dim3(COPY_THREADS), 0, (cudaStream_t)stream, 1, a); break;
                case 8: e = rg_launch(copy_pages_kernel<uint2>, grid, dim3(COPY_THREADS), 0, (cudaStream_t)stream, 1, a); break;
                case 4: e = rg_launch(copy_pages_kernel<unsigned>, grid, dim3(COPY_THREADS), 0, (cudaStream_t)stream, 1, a); break;
                case 2: e = rg_launch(copy_pages_kernel<unsigned short>, grid, dim3(COPY_THREADS), 0, (cudaStream_t)stream, 1, a); break;
                case 1: e = rg_launch(copy_pages_kernel<unsigned char>, grid, dim3(COPY_THREADS), 0, (cudaStream_t)stream, 1, a); break;
                default: return RG_ERR_UNSUPPORTED;
            }
            if (e) return e;
        }
    return 0;
}
