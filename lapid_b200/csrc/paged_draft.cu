// Drafted tokens over the paged cache: what a step makes of their parents, and what it keeps of them.
//
// tree    depth(t) = depth(parent) + 1, 0 without one; position = cached + depth; bit i of t: i is t or an ancestor of it (with a window: depth(t) - depth(i) < window).
//         A parent comes in front of its children, so a thread walks from its token to the root, setting bits on the way: a word is complete when the walk leaves it for
//         one further in front. Bound by latency: the record, the parents, a walk of as many shared loads as the token has ancestors: 8 trees of 16 tokens 3.3 to 3.5 us, 512 of up to 64 5.1 to 5.3.
// commit  keys and values at cached + path[i] go to cached + i, in every layer. Since path[i] >= i and the path rises, a thread that owns 16 bytes of a head and takes the path's
//         tokens in their order never overwrites what it has still to read. Pages that only rejected tokens lie in go back: the step's pages are the first ones of the
//         list, and are written there again, the kept ones first (requests in order), so that the caller drops the kept ones alone. Bound by latency, then by HBM: one request of 16 tokens in 32 layers 4.9 to 5.3 us, 32 of up to 24 10 to 12.6 us for 46 MB.
#include "common.cuh"
#include "paged.cuh"

namespace lb {

// A launch behind others of the stream
static void draft_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, dim3 grid, unsigned threads, bool pdl, cudaStream_t stream) {
    cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
}

// Whether the plan was made for this description; the first thread of the launch says so where not
__device__ __forceinline__ bool plan_fits(const uint32_t *stamped, uint32_t stamp, int *status) {
    const bool fits = *stamped == stamp;
    if (!fits && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && status) atomicOr(status, (int)PAGED_STATUS_PLAN);
    return fits;
}

// ------------------------------------------------------------------ tree
__global__ void __launch_bounds__(256) paged_tree_kernel(PagedTreeArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ int16_t parent[PAGED_TREE_MOST];
    const PagedShape &s = a.s;
    const int32_t words = (int32_t)s.tree;
    const bool fits = plan_fits(a.stamped, a.stamp, a.status);
    for (uint32_t r = blockIdx.x; r < s.requests; r += gridDim.x) {
        const uint4 x = ((const uint4 *)a.request)[r];
        const uint32_t n = fits ? min(x.y - x.x, PAGED_TREE_MOST) : 0, cached = x.z - n;
        bool bad = false;
        for (uint32_t t = threadIdx.x; t < n; t += blockDim.x) {
            const int32_t p = a.parents[x.x + t];
            bad |= p < -1 || p >= (int32_t)t;
            parent[t] = p >= 0 && p < (int32_t)t ? (int16_t)p : (int16_t)-1;  // (a token whose parent is none is a root)
        }
        if (bad && a.status) atomicOr(a.status, (int)PAGED_STATUS_INDEX);
        __syncthreads();
        for (uint32_t t = threadIdx.x; t < n; t += blockDim.x) {
            uint32_t *row = a.tree + (size_t)(x.x + t) * (1 + words), depth = 0, bits = 1u << (t & 31);
            int32_t w = (int32_t)t >> 5;
            for (int32_t i = w + 1; i < words; i++) row[1 + i] = 0;
            for (int32_t p = parent[t]; p >= 0; p = parent[p]) {
                depth++;
                if (s.window && depth >= s.window) continue;
                for (; p >> 5 < w; w--) row[1 + w] = bits, bits = 0;
                bits |= 1u << (p & 31);
            }
            for (; w >= 0; w--) row[1 + w] = bits, bits = 0;
            row[0] = depth;
            a.positions[x.x + t] = (int32_t)(cached + depth);
        }
        __syncthreads();
    }
}

cudaError_t launch_paged_tree(const PagedTreeArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    const uint32_t threads = a.s.max_new < 256 ? (a.s.max_new + 31) & ~31u : 256, most = (uint32_t)sm_count * 8;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    draft_config(cfg, attr, dim3(a.s.requests < most ? a.s.requests : most), threads, pdl, stream);
    return cudaLaunchKernelEx(&cfg, paged_tree_kernel, a);
}

// ------------------------------------------------------------------ commit
constexpr uint32_t COMMIT_THREADS = 128;

// How many tokens request r keeps: 0 where what it is told is out of range (`bad`)
__device__ __forceinline__ uint32_t accepted_of(const PagedCommitArgs &a, uint32_t r, uint32_t n, bool &bad) {
    const int32_t k = a.accepted[r];
    if (k >= 0 && (uint32_t)k <= n) return (uint32_t)k;
    bad = true;
    return 0;
}
// Entry i of a request's path rises from the one in front of it and stays among its tokens
__device__ __forceinline__ bool path_sound(const int32_t *path, uint32_t i, uint32_t n) {
    const int32_t p = path[i];
    return p >= 0 && (uint32_t)p < n && (i == 0 || path[i - 1] < p);
}

// Lengths, and the step's pages in the list: by one CTA, a thread a request. Where a page that the step needs is missing the list stays as it is and no request keeps anything.
__device__ void commit_pages(const PagedCommitArgs &a) {
    constexpr uint32_t WARPS = COMMIT_THREADS / 32;
    __shared__ uint32_t sums[2][WARPS];
    const PagedShape &s = a.s;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, shift = 31 - __clz(s.page);
    uint32_t all_kept = 0;  // over all requests
    bool missing = false;
    for (int pass = 0; pass < 2; pass++) {
        uint32_t kept = 0, back = 0;  // in front of this chunk
        for (uint32_t r0 = 0; r0 < s.requests; r0 += COMMIT_THREADS) {
            const uint32_t r = r0 + threadIdx.x;
            uint32_t have = 0, keep = 0, need = 0, end = 0, at_first = 0;
            bool lacks = false;
            if (r < s.requests) {
                const uint4 x = ((const uint4 *)a.request)[r];
                const uint32_t n = x.y - x.x, cached = x.z - n;
                at_first = cached;
                have = (cached + s.page - 1) >> shift, need = (x.z + s.page - 1) >> shift;
                const int32_t *const table = a.table + (size_t)r * s.max_blocks;
                auto page_of = [&](uint32_t b) -> uint32_t { return b >= need ? 0u : b < s.max_blocks ? (uint32_t)table[b] : ~0u; };
                const uint32_t page0 = page_of(have), page1 = page_of(have + 1);  // (asked for before the path is)
                bool bad = false;
                uint32_t k = accepted_of(a, r, n, bad);
                if (a.path)
                    for (uint32_t i = 0; i < k; i++) bad |= !path_sound(a.path + (size_t)r * s.max_new, i, n);
                if (bad) k = 0;
                if (bad && a.status) atomicOr(a.status, (int)PAGED_STATUS_INDEX);
                end = cached + k;
                keep = (end + s.page - 1) >> shift;
                lacks = page0 >= s.pages || page1 >= s.pages;
                for (uint32_t b = have + 2; b < need; b++) lacks |= page_of(b) >= s.pages;
            }
            uint32_t ki = keep - have, bi = need - keep;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, ki, o), v = __shfl_up_sync(0xffffffffu, bi, o);
                if (lane >= o) ki += u, bi += v;
            }
            __syncthreads();
            if (lane == 31) sums[0][warp] = ki, sums[1][warp] = bi;
            missing |= __syncthreads_or(lacks) != 0;
            uint32_t k_all = 0, b_all = 0, k_front = 0, b_front = 0;
#pragma unroll
            for (uint32_t w = 0; w < WARPS; w++) {
                if (w == warp) k_front = k_all, b_front = b_all;
                k_all += sums[0][w], b_all += sums[1][w];
            }
            if (s.requests <= COMMIT_THREADS) all_kept = k_all;
            if (r < s.requests && (pass || s.requests <= COMMIT_THREADS)) {
                uint32_t to_kept = kept + k_front + ki - (keep - have), to_back = all_kept + back + b_front + bi - (need - keep);
                a.kv_lens[r] = (int32_t)(missing ? at_first : end);
                for (uint32_t b = have; b < need && !missing; b++) {
                    const uint32_t to = b < keep ? to_kept++ : to_back++;
                    if (to < a.n_free) a.free_pages[to] = a.table[(size_t)r * s.max_blocks + b];
                }
            }
            kept += k_all, back += b_all;
        }
        all_kept = kept;
        if (s.requests <= COMMIT_THREADS) break;
    }
    if (threadIdx.x == 0) *a.used = missing ? 0 : (int32_t)all_kept;
}

// A CTA has one request and some of the caches: where its tokens lie and where they go is found once, in shared memory, and what is asked for first (record, accepted, path) does not wait for each other.
// blockIdx.x: a group of caches, and behind them (where the launch has pages) one CTA for the lengths and pages; blockIdx.y walks the requests
__global__ void __launch_bounds__(COMMIT_THREADS) paged_commit_kernel(const __grid_constant__ PagedCommitArgs a, uint32_t each) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr uint32_t NONE = ~0u, B = 4;  // tokens whose bytes are in flight
    __shared__ uint32_t from[PAGED_TREE_MOST], to[PAGED_TREE_MOST];  // rows of a cache, of the first head
    const PagedShape &s = a.s;
    const uint32_t groups = (a.caches + each - 1) / each;
    if (!plan_fits(a.stamped, a.stamp, a.status)) return;
    if (blockIdx.x == groups) {
        if (blockIdx.y == 0) commit_pages(a);
        return;
    }
    const uint32_t shift = 31 - __clz(s.page), chunks = s.d / 8, columns = s.hkv * chunks;
    for (uint32_t r = blockIdx.y; r < s.requests; r += gridDim.y) {
        const int32_t *const path = a.path + (size_t)r * s.max_new, *const table = a.table + (size_t)r * s.max_blocks;
        const int32_t mine = threadIdx.x < s.max_new ? path[threadIdx.x] : -1, before = threadIdx.x && threadIdx.x < s.max_new ? path[threadIdx.x - 1] : -1;
        const uint4 x = ((const uint4 *)a.request)[r];
        const uint32_t n = x.y - x.x, cached = x.z - n;
        bool bad = false;
        const uint32_t k = accepted_of(a, r, n, bad);
        if (threadIdx.x < k) bad |= mine < 0 || (uint32_t)mine >= n || (threadIdx.x && before >= mine);
        for (uint32_t i = threadIdx.x + COMMIT_THREADS; i < k; i += COMMIT_THREADS) bad |= !path_sound(path, i, n);
        auto row_of = [&](uint32_t token) -> uint32_t {
            const uint32_t pos = cached + token, block = pos >> shift;
            const int32_t page = block < s.max_blocks ? table[block] : -1;
            if (page >= 0 && (uint32_t)page < s.pages) return (uint32_t)page * s.hkv * s.page + (pos & (s.page - 1));
            if (a.status) atomicOr(a.status, (int)PAGED_STATUS_INDEX);
            return NONE;
        };
        if (__syncthreads_or(bad)) continue;  // (the pages' CTA tells of it)
        for (uint32_t i = threadIdx.x; i < k; i += COMMIT_THREADS) {
            const uint32_t src = (uint32_t)(i == threadIdx.x ? mine : path[i]);
            uint32_t f = NONE, t = NONE;
            if (src != i) f = row_of(src), t = row_of(i);
            from[i] = f, to[i] = f == NONE ? NONE : t;
        }
        __syncthreads();
        // a thread has 16 bytes of a head, and takes the tokens in their order
        const uint32_t first = blockIdx.x * each, count = min(each, a.caches - first);
        for (uint32_t c = threadIdx.x; c < columns * count; c += COMMIT_THREADS) {
            const uint32_t cache = c / columns, col = c - cache * columns, head = col / chunks;
            uint4 *const base = (uint4 *)a.cache[first + cache] + (size_t)head * s.page * chunks + (col - head * chunks);
            for (uint32_t i0 = 0; i0 < k; i0 += B) {
                uint4 v[B];
                uint32_t at[B];
#pragma unroll
                for (uint32_t i = 0; i < B; i++) {
                    at[i] = i0 + i < k ? to[i0 + i] : NONE;
                    if (at[i] != NONE) v[i] = base[(size_t)from[i0 + i] * chunks];
                }
#pragma unroll
                for (uint32_t i = 0; i < B; i++)
                    if (at[i] != NONE) base[(size_t)at[i] * chunks] = v[i];
            }
        }
        __syncthreads();  // (the rows are read)
    }
}

cudaError_t launch_paged_commit(const PagedCommitArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    // caches for each CTA: one, or as many as leave some eight CTAs an SM
    const uint64_t all = (uint64_t)a.caches * a.s.requests, most = 8 * (uint64_t)sm_count;
    const uint32_t each = (uint32_t)(all > most ? (all + most - 1) / most : 1), groups = (a.caches + each - 1) / each;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    draft_config(cfg, attr, dim3(groups + (a.pages ? 1 : 0), a.s.requests < 65535 ? (a.s.requests ? a.s.requests : 1) : 65535), COMMIT_THREADS, pdl, stream);
    return cudaLaunchKernelEx(&cfg, paged_commit_kernel, a, each);
}

}  // namespace lb
