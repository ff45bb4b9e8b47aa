// The paged key/value cache: block tables and slot maps from the requests' lengths, and the append of new keys and values.
//
// plan    start[r] = sum of the new lengths before r (those within bounds, whether their request takes part or not), first[r] = sum of the pages taken
//         before r; token t of r lies at position cached + t, in block pos / page of its table row, slot = table[r][block] * page + pos % page.
//         New blocks take the pages free_pages[first[r]...] in the requests' order, so the result does not depend on timing. The plan also cuts the
//         work of the attention launches that follow (paged.cuh): which request, head, tile and step each CTA begins with. That is
//         done once a step, and every layer's launch reads it.
//         What bounds it is latency: one launch, two scans over the requests, a search a token and a search a start. Every CTA scans the
//         lengths itself so that nothing passes between CTAs, and takes its share of the tokens, blocks and starts. 64 requests of one token 4.2 us, 48
//         prompts (65520 tokens) 7.8, 256 requests 9.1, 1024 9.1. Above that one CTA makes all starts, from prefixes in global memory: 1025 requests 36 us, 2048 38.
// append  (x, y) -> (x cos - y sin, y cos + x sin) in f32 for the rotary pairs of q and k, one rounding to the cache's type; k and v go
//         to their slots. Bound by memory: each element is read once and written once; a thread keeps the angles of its
//         four pairs in registers over the heads of a token.
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged.cuh"

namespace lb {

// ------------------------------------------------------------------ layout of a plan (host)
static uint32_t words_up(uint32_t w) { return (w + 63) & ~63u; }

uint32_t paged_part_floats(const PagedShape &s, uint32_t rows) { return rows * ((s.d > 64 ? 128 : 64) + 2); }

PagedPlanLayout paged_plan_layout(const PagedShape &s) {
    PagedPlanLayout l{};
    uint32_t w = 0;
    auto take = [&](uint32_t n) {
        const uint32_t at = w;
        w = words_up(w + n);
        return at;
    };
    const uint32_t cs = paged_attn_small_ctas(PAGED_MAX_SMS), cl = paged_has_large(s) ? paged_attn_large_ctas(PAGED_MAX_SMS) : 0;
    l.past = take(1);  // (the first word: written before it is known whether the plan is one for this description)
    l.request = take(4 * s.requests);
    l.units_small = take(s.requests + 1);
    l.units_large = take(s.requests + 1);
    l.start_small = take(sizeof(PagedStart) / 4 * cs);
    l.start_large = take(sizeof(PagedStart) / 4 * cl);
    l.count_small = take(cs);
    l.count_large = take(2 * cl);  // (for each of a tile's two halves)
    l.part_small = (size_t)w * 4;
    l.part_large = l.part_small + (size_t)cs * 2 * paged_part_floats(s, PAGED_SMALL_ROWS) * 4;
    l.bytes = l.part_large + (size_t)cl * 2 * paged_part_floats(s, PAGED_LARGE_ROWS) * 4;
    return l;
}

bool paged_has_large(const PagedShape &s) { return !paged_is_small(s, s.max_new); }

uint32_t paged_stamp(const PagedShape &s) {
    uint32_t h = 2166136261u;  // (Fowler, Noll and Vo's hash over the words a plan depends on)
    for (uint32_t v : {s.g, s.hkv, s.page, s.requests, s.tokens, s.max_blocks, s.max_new, s.mask, s.window, s.d > 64 ? 128u : 64u, s.tree})
        for (int b = 0; b < 4; b++) h = (h ^ ((v >> (8 * b)) & 0xff)) * 16777619u;
    return h | 1u;  // never what a zeroed buffer holds
}

// ------------------------------------------------------------------ plan
// T threads take T requests at a time: 256 where there are no more (64 requests: 4.2 us, with 1024 threads and a scan for each sum 6.7), else 1024.
template <uint32_t T> struct PlanShared {
    uint64_t warp_sum[T / 32];
    uint32_t end_pages;  // pages taken in front of the request whose rows pass the last one
    uint32_t start[T], n[T], first[T], cached[T], have[T], kv[T];  // n: tokens that take part
    uint32_t small[T + 1], large[T + 1];    // units before the request
    uint32_t tiles[T + 1], steps[T];        // of many rows: tiles before the request, units of its tiles for one head
};

// Two sums at once (low and high half) over the threads before this one; `total`: over all
template <uint32_t T> __device__ __forceinline__ uint64_t block_scan(uint64_t v, PlanShared<T> &sh, uint64_t &total) {
    constexpr uint32_t WARPS = T / 32;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    __syncthreads();  // the sums of the scan before have been read
    if (lane == 31) sh.warp_sum[warp] = inc;
    __syncthreads();
    uint64_t w = lane < WARPS ? sh.warp_sum[lane] : 0, winc = w;
#pragma unroll
    for (int o = 1; o < (int)WARPS; o <<= 1) {
        const uint64_t x = __shfl_up_sync(0xffffffffu, winc, o);
        if (lane >= o) winc += x;
    }
    total = __shfl_sync(0xffffffffu, winc, WARPS - 1);
    return __shfl_sync(0xffffffffu, winc - w, warp) + inc - v;
}
__device__ __forceinline__ uint64_t both(uint32_t lo, uint32_t hi) { return lo | (uint64_t)hi << 32; }

// The last i < n with a[i] <= x (a rises, a[0] <= x)
__device__ __forceinline__ uint32_t last_at_most(const uint32_t *a, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// What each CTA of an attention launch begins with: warp `worker` of `workers` takes every workers-th of them. `prefix`: units before each request, `request`: what the
// plan holds of one.
template <class Request>
__device__ void cut_units(const PagedPlanArgs &a, uint32_t units, uint32_t ctas, uint32_t all, const uint32_t *prefix, Request request, uint32_t *starts, uint32_t rows, uint32_t keys,
                          uint32_t extra, uint32_t worker, uint32_t workers) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t b = worker; b < all; b += workers) {
        PagedStart x{};
        x.stamp = a.stamp, x.units = units, x.ctas = ctas;
        if (b < ctas) {
            x.u0 = paged_span(units, ctas, b + (lane & 1));  // (an even lane: where the span begins, an odd one: where it ends)
            x.u1 = __shfl_sync(0xffffffffu, x.u0, 1);
            x.u0 = __shfl_sync(0xffffffffu, x.u0, 0);
            const uint32_t r = last_at_most(prefix, a.s.requests, x.u0);
            const uint4 q = request(r);
            x.r = r, x.q0 = q.x, x.n = q.y - q.x, x.kv = q.z;
            const uint32_t per_head = (prefix[r + 1] - prefix[r]) / a.s.hkv, off = x.u0 - prefix[r], tiles = paged_tiles(a.s, x.n, rows);
            x.head = off / per_head;
            uint32_t rem = off - x.head * per_head;
            for (uint32_t i0 = 0; i0 < tiles; i0 += 32) {
                const uint32_t mine = i0 + lane < tiles ? paged_tile(a.s, x.n, x.kv, i0 + lane, rows, keys).steps + extra : 0;
                uint32_t inc = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                const uint32_t behind = __ballot_sync(0xffffffffu, inc > rem);
                if (behind) {
                    const int who = __ffs(behind) - 1;
                    x.tile = i0 + who;
                    rem -= __shfl_sync(0xffffffffu, inc - mine, who);
                    break;
                }
                rem -= __shfl_sync(0xffffffffu, inc, 31);
            }
            x.place = rem;
        }
        if (lane < 3) {
            uint4 v = make_uint4(x.stamp, x.units, x.ctas, x.u0);
            if (lane == 1) v = make_uint4(x.u1, x.r, x.head, x.tile);
            if (lane == 2) v = make_uint4(x.place, x.q0, x.n, x.kv);
            ((uint4 *)starts)[b * (sizeof(PagedStart) / 16) + lane] = v;
        }
    }
}

template <uint32_t T> __global__ void __launch_bounds__(T) paged_plan_kernel(PagedPlanArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ PlanShared<T> sh;
    const PagedShape &s = a.s;
    const uint32_t tid = threadIdx.x, worker = blockIdx.x, workers = gridDim.x, shift = 31 - __clz(s.page);  // (page sizes are powers of two)
    const bool one = s.requests <= T;  // chunk: what the searches for the starts need stays in shared memory
    const bool counts = one || blockIdx.x == 0, writes = blockIdx.x == 0;
    uint32_t base = 0, taken = 0, small = 0, large = 0;  // tokens, pages and units of the chunks before
    uint32_t bad = 0;
    for (uint32_t r0 = 0; r0 < s.requests; r0 += T) {
        const uint32_t r = r0 + tid, count = min(T, s.requests - r0);
        uint32_t own = 0, n = 0, c = 0, have = 0, need = 0;  // rows of q, new tokens
        if (r < s.requests) {
            const int32_t n0 = a.new_lens[r], c0 = a.cached[r];
            const uint64_t blocks = ((uint64_t)(uint32_t)c0 + (s.mask == PAGED_CROSS ? 0u : (uint32_t)n0) + s.page - 1) >> shift;
            const bool counted = n0 >= 0 && (uint32_t)n0 <= s.max_new;
            c = (uint32_t)c0;
            if (counted) own = (uint32_t)n0;
            if (!counted || c0 < 0 || blocks > s.max_blocks) {
                bad |= PAGED_STATUS_LENGTHS;  // such a request takes no part: it keeps the length that it has, and its rows, so that the others' stay where they are
            } else {
                n = own;
                have = (c + s.page - 1) >> shift;
                need = (uint32_t)blocks;
            }
        }
        if (tid == 0) sh.end_pages = ~0u;
        uint64_t total;
        uint64_t at = block_scan<T>(both(own, need - have), sh, total);
        const uint64_t pages = total;  // (high half)
        const uint32_t at_n = base + (uint32_t)at, at_p = taken + (uint32_t)(at >> 32), lo = min(at_n, s.tokens), end_n = min(base + (uint32_t)total, s.tokens);
        // A request whose rows pass the last one of q takes no part either, and none behind it has rows: the pages end where it stands.
        if (n && at_n + n > s.tokens) bad |= PAGED_STATUS_LENGTHS, n = 0;
        if (at_n <= s.tokens && at_n + own > s.tokens) sh.end_pages = at_p;
        const uint32_t kv = s.mask == PAGED_CROSS ? c : c + n;
        sh.start[tid] = lo;
        sh.n[tid] = n;
        sh.first[tid] = at_p;
        sh.cached[tid] = c;
        sh.have[tid] = have;
        sh.kv[tid] = kv;
        if (counts) {
            const bool few = paged_is_small(s, n);
            uint32_t us = 0, ul = 0;
            if (few && n)
                for (uint32_t i = 0; i < paged_tiles(s, n, PAGED_SMALL_ROWS); i++) us += paged_tile(s, n, kv, i, PAGED_SMALL_ROWS, PAGED_SMALL_KEYS).steps;
            if (a.ctas_large) {  // all tiles of many rows, a thread each (they add whole numbers: in whatever order)
                const uint32_t rows = paged_large_rows(s), tiles = few ? 0 : paged_tiles(s, n, rows);
                const uint32_t before = (uint32_t)block_scan<T>(tiles, sh, total);
                sh.tiles[tid] = before;
                sh.steps[tid] = 0;
                if (tid == 0) sh.tiles[count] = (uint32_t)total;
                __syncthreads();
                for (uint32_t i = tid; i < (uint32_t)total; i += T) {
                    const uint32_t q = last_at_most(sh.tiles, count, i);
                    atomicAdd(&sh.steps[q], paged_tile(s, sh.n[q], sh.kv[q], i - sh.tiles[q], rows, s.large_keys).steps + PAGED_LARGE_EXTRA);
                }
                __syncthreads();
                ul = sh.steps[tid];
            }
            at = block_scan<T>(both(us * s.hkv, ul * s.hkv), sh, total);
            sh.small[tid] = small + (uint32_t)at, sh.large[tid] = large + (uint32_t)(at >> 32);
            small += (uint32_t)total, large += (uint32_t)(total >> 32);
            if (tid == 0) sh.small[count] = small, sh.large[count] = large;
        }
        if (writes && r < s.requests) {
            ((uint4 *)(a.plan + a.l.request))[r] = make_uint4(lo, lo + n, kv, 0);
            a.kv_lens[r] = (int32_t)kv;
            if (!one) a.plan[a.l.units_small + r] = sh.small[tid], a.plan[a.l.units_large + r] = sh.large[tid];
        }
        __syncthreads();
        const uint32_t end_p = min(taken + (uint32_t)(pages >> 32), sh.end_pages);
        for (uint32_t j = taken + worker * T + tid; j < end_p; j += workers * T) {
            const uint32_t i = last_at_most(sh.first, count, j);
            int32_t page = -1;
            // (the list ends at n_free, or in entries below 0 where only the device knows its length)
            if (j >= a.n_free) bad |= PAGED_STATUS_PAGES;
            else if ((page = a.free_pages[j]) < 0 || (uint32_t)page >= s.pages) bad |= page < 0 ? PAGED_STATUS_PAGES : PAGED_STATUS_INDEX, page = -1;
            a.table[(size_t)(r0 + i) * s.max_blocks + sh.have[i] + (j - sh.first[i])] = page;
        }
        // (the last CTA begins: the first one has the pages)
        for (uint32_t t = base + (workers - 1 - worker) * T + tid; t < end_n; t += workers * T) {
            const uint32_t i = last_at_most(sh.start, count, t), pos = sh.cached[i] + (t - sh.start[i]), block = pos >> shift;
            const bool part = t - sh.start[i] < sh.n[i];
            int32_t slot = -1;
            if (part && s.mask != PAGED_CROSS) {
                int32_t page = -1;
                if (block < sh.have[i]) page = a.table[(size_t)(r0 + i) * s.max_blocks + block];
                else if (sh.first[i] + (block - sh.have[i]) < a.n_free) page = a.free_pages[sh.first[i] + (block - sh.have[i])];
                if (page >= 0 && (uint32_t)page < s.pages) slot = (int32_t)(((uint32_t)page << shift) + (pos & (s.page - 1)));
                else if (block < sh.have[i]) bad |= PAGED_STATUS_INDEX;
            }
            a.slots[t] = slot;
            a.positions[t] = part ? (int32_t)pos : -1;
        }
        base = end_n;
        taken = end_p;
        if (!one) __syncthreads();  // the tables of this chunk are read
    }
    for (uint32_t t = base + worker * T + tid; t < s.tokens; t += workers * T) a.slots[t] = a.positions[t] = -1;
    if (bad && a.status) atomicOr(a.status, (int)bad);
    if (writes) {
        if (tid == 0) {
            *a.used = (int32_t)taken;
            a.plan[a.l.past] = 0;
            if (!one) a.plan[a.l.units_small + s.requests] = small, a.plan[a.l.units_large + s.requests] = large;
        }
        for (uint32_t b = tid; b < a.ctas_small; b += T) a.plan[a.l.count_small + b] = 0;
        for (uint32_t b = tid; b < 2 * a.ctas_large; b += T) a.plan[a.l.count_large + b] = 0;
    }
    if (!counts) return;
    if (!one) __syncthreads();  // (the tables in the plan are read)
    // Few rows: a step a CTA where every CTA then has an SM of its own, else two. (One token over 48, 192, 512, 1024 keys and 8 heads: with a step 5.7, 6.7, 6.9, 7.4 us, with
    // two 7.5, 10.5, 7.7, 9.4, over 128 keys 6.7 and 5.8; over 4096 keys, where there are more steps than SMs, 11.5 and 10.5.)
    uint32_t cs = small <= a.ctas_small / 2 ? small : min((small + 1) / 2, a.ctas_small);
    uint32_t cl = large < a.ctas_large * PAGED_LARGE_MIN ? (large + PAGED_LARGE_MIN - 1) / PAGED_LARGE_MIN : a.ctas_large;
    if (small && large) {
        // Both kernels have work, one bound by memory, the other by its products: they run side by side, on as many SMs as their shares of the work
        // (a chunk of 512 tokens beside 11 tokens of other requests, 3000 keys each: one after the other 83 us, side by side 62). Every CTA of the kernel for many rows holds an SM; the other's come, two to an SM,
        // where one of those had nothing to do.
        const uint64_t ts = (uint64_t)small * (s.d > 64 ? PAGED_SMALL_NS_128 : PAGED_SMALL_NS_64), tl = (uint64_t)large * (s.d > 64 ? PAGED_LARGE_NS_128 : PAGED_LARGE_NS_64);
        const uint32_t sms = a.ctas_large, share = (uint32_t)(sms * tl / (ts + tl));
        cl = min(cl, max(share, 1u));
        cs = min(cs, max(a.ctas_small / sms * (sms - cl), 1u));
    }
    auto request = [&](uint32_t r) { return one ? make_uint4(sh.start[r], sh.start[r] + sh.n[r], sh.kv[r], 0) : ((const uint4 *)(a.plan + a.l.request))[r]; };
    const uint32_t warp = worker * (T / 32) + tid / 32, warps = (one ? workers : 1) * (T / 32);
    cut_units(a, small, cs, a.ctas_small, one ? sh.small : a.plan + a.l.units_small, request, a.plan + a.l.start_small, PAGED_SMALL_ROWS, PAGED_SMALL_KEYS, 0, warp, warps);
    // (from the other end: a warp has a start of one kind or of the other)
    if (a.ctas_large)
        cut_units(a, large, cl, a.ctas_large, one ? sh.large : a.plan + a.l.units_large, request, a.plan + a.l.start_large, paged_large_rows(s), s.large_keys, PAGED_LARGE_EXTRA, warps - 1 - warp, warps);
}

static void paged_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, dim3 grid, unsigned threads, size_t smem, bool pdl, cudaStream_t stream) {
    cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
}

cudaError_t launch_paged_plan(const PagedPlanArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    const uint32_t T = a.s.requests <= 256 ? 256 : 1024;
    // a thread for each token, a warp for each start
    const uint32_t starts = (a.ctas_small + a.ctas_large + T / 32 - 1) / (T / 32), tokens = (a.s.tokens + T - 1) / T, want = starts > tokens ? starts : tokens;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    paged_config(cfg, attr, dim3(want < (uint32_t)sm_count ? want : (uint32_t)sm_count), T, 0, pdl, stream);
    return T == 256 ? cudaLaunchKernelEx(&cfg, paged_plan_kernel<256>, a) : cudaLaunchKernelEx(&cfg, paged_plan_kernel<1024>, a);
}

// ------------------------------------------------------------------ append
// Heads whose loads a thread has in flight. 8192 tokens of 48 heads of 128: 47.6 us (0.98 of the measured bandwidth); CTAs of 256 threads 52.8, of 64 49.1, two heads 48.2,
// four 49.1; with the rows asked for behind slot and position 61. From f16 or bf16 rows 51.7 for two thirds of the bytes (31.5 us of bandwidth): as many requests, half of the bytes in each.
constexpr uint32_t APPEND_THREADS = 128, APPEND_HEADS = 3;

__device__ __forceinline__ uint32_t pack_half(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *(const uint32_t *)&r;
    }
    const __half2 r = __floats2half2_rn(a, b);
    return *(const uint32_t *)&r;
}
// four elements from `i` on of the row at `row`
template <int SRC, bool VEC> __device__ __forceinline__ float4 load4(const void *row, uint32_t i) {
    if constexpr (!VEC) return make_float4(load_act(row, i, SRC), load_act(row, i + 1, SRC), load_act(row, i + 2, SRC), load_act(row, i + 3, SRC));
    else if constexpr (SRC == ACT_F32) return *(const float4 *)((const float *)row + i);
    else {
        const uint2 w = *(const uint2 *)((const unsigned short *)row + i);
        return make_float4(widen_act(w.x & 0xffff, SRC), widen_act(w.x >> 16, SRC), widen_act(w.y & 0xffff, SRC), widen_act(w.y >> 16, SRC));
    }
}

// blockIdx.x walks the tokens, blockIdx.y takes every gridDim.y-th batch of heads. A thread owns eight elements of a head: the rotary pairs
// (i, i + rot / 2), i = 4 c..4 c + 3 (halves), or the neighbours (2 i, 2 i + 1) of the same i, or eight elements as they are. VEC: the rows allow loads of four elements.
template <int SRC, bool VEC> __global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(PagedAppendArgs p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const PagedShape &s = p.s;
    const uint32_t chunks = s.d / 8, lanes = APPEND_THREADS / chunks, c = threadIdx.x % chunks, hl = threadIdx.x / chunks;
    if (hl >= lanes) return;
    const uint32_t hq = p.q ? s.hq : 0, heads = hq + (p.k ? 2 * s.hkv : 0), half = p.rot / 2;
    const bool turned = c < p.rot / 8;
    const bool bf16 = s.bf16;
    const uint32_t shift = 31 - __clz(s.page);  // (page sizes are powers of two)
    for (uint32_t t = blockIdx.x; t < s.tokens; t += gridDim.x) {
        const int32_t slot = p.slots ? p.slots[t] : -1, pos = p.positions[t];
        float4 cs = make_float4(1.0f, 1.0f, 1.0f, 1.0f), sn = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const bool stored = slot >= 0 && (uint32_t)slot < s.pages << shift, sound = pos >= 0 && !(p.rot && (uint32_t)pos >= p.rope_rows) && (slot == -1 || stored);
        bool first = true;
        for (uint32_t h0 = blockIdx.y * lanes * APPEND_HEADS; h0 < heads; h0 += gridDim.y * lanes * APPEND_HEADS) {
            // (the rows do not wait for the slot and the position)
            float4 x[APPEND_HEADS], y[APPEND_HEADS];
#pragma unroll
            for (uint32_t j = 0; j < APPEND_HEADS; j++) {
                const uint32_t h = h0 + j * lanes + hl;
                if (h >= heads) continue;
                const bool is_q = h < hq, is_v = h >= hq + s.hkv;
                const PagedView &w = is_q ? p.qv : is_v ? p.vv : p.kv;
                const uint32_t hh = is_q ? h : is_v ? h - hq - s.hkv : h - hq;
                const void *base = is_q ? p.q : is_v ? p.v : p.k;
                const void *row = (const char *)base + (w.off + (uint64_t)t * w.token + (uint64_t)hh * w.head) * act_elem_bytes(SRC);
                const bool split = turned && !is_v && !p.neighbours;
                x[j] = load4<SRC, VEC>(row, split ? 4 * c : 8 * c);
                y[j] = load4<SRC, VEC>(row, split ? 4 * c + half : 8 * c + 4);
            }
            if (!sound) break;
            if (first && turned) {
                cs = *(const float4 *)(p.rope + (size_t)pos * p.rot + 4 * c);
                sn = *(const float4 *)(p.rope + (size_t)pos * p.rot + half + 4 * c);
            }
            first = false;
            const uint32_t page = (uint32_t)slot >> shift, in_page = (uint32_t)slot & (s.page - 1);
#pragma unroll
            for (uint32_t j = 0; j < APPEND_HEADS; j++) {
                const uint32_t h = h0 + j * lanes + hl;
                if (h >= heads) continue;
                const bool is_q = h < hq, is_v = h >= hq + s.hkv;
                if (!is_q && !stored) continue;
                const uint32_t hh = is_q ? h : is_v ? h - hq - s.hkv : h - hq;
                uint16_t *row = is_q ? (uint16_t *)p.q_out + ((size_t)t * s.hq + hh) * s.d
                                     : (uint16_t *)(is_v ? p.v_cache : p.k_cache) + (((size_t)page * s.hkv + hh) * s.page + in_page) * s.d;
                const float4 u = x[j], v = y[j];
                if (turned && !is_v && !p.neighbours) {
                    const uint2 lo = make_uint2(pack_half(fmaf(u.x, cs.x, -v.x * sn.x), fmaf(u.y, cs.y, -v.y * sn.y), bf16),
                                                pack_half(fmaf(u.z, cs.z, -v.z * sn.z), fmaf(u.w, cs.w, -v.w * sn.w), bf16));
                    const uint2 hi = make_uint2(pack_half(fmaf(v.x, cs.x, u.x * sn.x), fmaf(v.y, cs.y, u.y * sn.y), bf16),
                                                pack_half(fmaf(v.z, cs.z, u.z * sn.z), fmaf(v.w, cs.w, u.w * sn.w), bf16));
                    *(uint2 *)(row + 4 * c) = lo;
                    *(uint2 *)(row + 4 * c + half) = hi;
                } else if (turned && !is_v) {
                    *(uint4 *)(row + 8 * c) = make_uint4(pack_half(fmaf(u.x, cs.x, -u.y * sn.x), fmaf(u.y, cs.x, u.x * sn.x), bf16),
                                                         pack_half(fmaf(u.z, cs.y, -u.w * sn.y), fmaf(u.w, cs.y, u.z * sn.y), bf16),
                                                         pack_half(fmaf(v.x, cs.z, -v.y * sn.z), fmaf(v.y, cs.z, v.x * sn.z), bf16),
                                                         pack_half(fmaf(v.z, cs.w, -v.w * sn.w), fmaf(v.w, cs.w, v.z * sn.w), bf16));
                } else {
                    *(uint4 *)(row + 8 * c) = make_uint4(pack_half(u.x, u.y, bf16), pack_half(u.z, u.w, bf16), pack_half(v.x, v.y, bf16), pack_half(v.z, v.w, bf16));
                }
            }
        }
        if (!sound && pos != -1 && threadIdx.x == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_INDEX);
    }
}

template <int SRC> static cudaError_t append_src(const PagedAppendArgs &a, bool vec, const cudaLaunchConfig_t &cfg) {
    return vec ? cudaLaunchKernelEx(&cfg, paged_append_kernel<SRC, true>, a) : cudaLaunchKernelEx(&cfg, paged_append_kernel<SRC, false>, a);
}

cudaError_t launch_paged_append(const PagedAppendArgs &a, bool pdl, cudaStream_t stream) {
    const uint32_t eb = act_elem_bytes(a.src_type), per = APPEND_THREADS / (a.s.d / 8) * APPEND_HEADS, heads = (a.q ? a.s.hq : 0) + (a.k ? 2 * a.s.hkv : 0);
    bool vec = true;  // every group of four elements starts on a multiple of its size
    auto check = [&](const void *base, const PagedView &v) {
        if (base && (((uintptr_t)base + v.off * eb) % (4 * eb) || v.head % 4 || v.token % 4)) vec = false;
    };
    check(a.q, a.qv);
    check(a.k, a.kv);
    check(a.v, a.vv);
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    // few tokens: a CTA for each batch of heads; many: one CTA walks a token's heads and keeps its angles
    const uint32_t batches = (heads + per - 1) / per;
    paged_config(cfg, attr, dim3(a.s.tokens < (1u << 20) ? a.s.tokens : 1u << 20, a.s.tokens < 512 ? batches : 1), APPEND_THREADS, 0, pdl, stream);
    return a.src_type == ACT_F32 ? append_src<ACT_F32>(a, vec, cfg) : a.src_type == ACT_F16 ? append_src<ACT_F16>(a, vec, cfg) : append_src<ACT_BF16>(a, vec, cfg);
}

}  // namespace lb
