// Attention over the pages for requests of few rows: single tokens, a few speculated ones, short chunks.
//
//   s = scale q k^T over the keys that the mask leaves a row;  m = max s, p = exp(s - m), l = sum p, out = sum p v / l
//
// in one pass over the keys: m, l and the accumulator are rescaled when m grows. What bounds it is HBM: every key and value is read once
// for the g query heads that share it (g x 2 operations a byte), so the query heads of one key/value head are the 16 rows of `mma.sync.m16n8k16`
// -- the operands it multiplies come straight from the copied pages, and the results are where the next product wants them; the
// tensor-memory instruction would want 128 rows and its softmax weights back in tensor memory.
//
// The steps (64 keys of one tile) of all requests and heads are one sequence, cut into equal spans, one a CTA (paged.cuh): requests of any
// lengths keep every SM busy to the end. A producer warp fills a ring of steps with TMA copies of (parts of) pages, four warps take 16
// keys of every step each, with maxima, sums and accumulators of their own, which meet at the end of a tile. A tile that a span's end
// cuts is left in the plan buffer by each of its CTAs; the one that comes last adds the pieces up, in the order of the keys.
//
// Measured: 64 requests of one token over 820 to 8192 keys, 32 query and 8 key heads of 128, 187 us for 1.18 GB (6.3 TB/s, 0.96 of the measured copy rate); two over 118 to
// 131 thousand keys, 64 query heads, 165 us (0.94); one over 4096 keys 10.5 us, of which 2.6 are its bytes: four trips to memory one after the other
// (start, page number, page, pieces of the other CTAs) and the launch. Two CTAs of 110 KB an SM: one's end is the other's work.
#include <cuda.h>
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "pipe.cuh"

namespace lb {

namespace pa {

using namespace pipe;

constexpr int KEYS = PAGED_SMALL_KEYS, ROWS = PAGED_SMALL_ROWS;
constexpr int WARPS = 4, THREADS = 32 * (WARPS + 1);  // and the producer
constexpr int CHUNK = 32, MEET = WARPS * ROWS * (CHUNK + 8);  // the accumulators meet in shared memory 32 columns of 16 rows at a time, or more of fewer; the pitch avoids bank conflicts
constexpr uint32_t SPIN_LIMIT = 1u << 19;            // a wait gives up after so many attempts, each as long as the hardware lets one sleep

template <int DP> struct Cfg {
    static constexpr int HALVES = DP / 64;                  // a copied row is 64 elements wide: the width of a 128-byte swizzled row
    static constexpr int PART = KEYS * 128;                 // bytes of one half of a step's keys (or values)
    static constexpr int STAGE = 2 * HALVES * PART;
    static constexpr int STAGES = 3 * 128 / DP;
    static constexpr int SMEM = STAGES * STAGE + MEET * 4 + 2 * WARPS * ROWS * 4 + 16 * STAGES + 16 + 1024;
};

template <bool BF16> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS> __device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool BF16> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); }

// Where a CTA is in the sequence of steps
struct Walk {
    uint32_t r, head, tile, tiles, n, kv, q0;
    PagedTile t;
};
__device__ __forceinline__ void load_request(const PagedAttnArgs &p, Walk &w) {
    const uint4 x = ((const uint4 *)(p.plan + p.l.request))[w.r];
    w.q0 = x.x, w.n = x.y - x.x, w.kv = x.z;
    w.tiles = paged_tiles(p.s, w.n, ROWS);
}
__device__ __forceinline__ void load_tile(const PagedAttnArgs &p, Walk &w) { w.t = paged_tile(p.s, w.n, w.kv, w.tile, ROWS, KEYS); }
__device__ __forceinline__ void next_tile(const PagedAttnArgs &p, Walk &w) {
    if (++w.tile == w.tiles) {
        w.tile = 0;
        if (++w.head == p.s.hkv) {
            w.head = 0;
            do {
                w.r++;
                load_request(p, w);
            } while (w.n == 0 || !paged_is_small(p.s, w.n));
        }
    }
    load_tile(p, w);
}

__device__ __forceinline__ void store_half4(unsigned short *row, uint32_t col, uint32_t d, float4 v, bool bf16, bool vec) {
    if (vec && col + 4 <= d) {
        *(uint2 *)(row + col) = bf16 ? make_uint2(pack<true>(v.x, v.y), pack<true>(v.z, v.w)) : make_uint2(pack<false>(v.x, v.y), pack<false>(v.z, v.w));
        return;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        if (col + i < d) row[col + i] = (unsigned short)(bf16 ? pack<true>(f[i], 0.0f) : pack<false>(f[i], 0.0f));
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(THREADS, 2) paged_attn_small_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, PagedAttnArgs p) {
    using C = Cfg<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((0u - s32(smem_raw)) & 1023u);
    float *meet = (float *)(smem + C::STAGES * C::STAGE);                  // [warp][row][columns]
    float *meet_m = meet + MEET, *meet_l = meet_m + WARPS * ROWS;
    uint64_t *full = (uint64_t *)(meet_l + WARPS * ROWS), *empty = full + C::STAGES;
    volatile uint32_t *is_last = (volatile uint32_t *)(empty + C::STAGES);
    const PagedShape &s = p.s;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, WARPS);
        }
        mbar_fence_init();
    }
    // Behind the kernel for many rows this one starts as soon as all that was in front of that is over; the two share no memory that either writes. That what was in front is
    // visible here comes through a word that the other's first CTA releases behind its own wait; where it is not there the wait for that kernel's end does it.
    // And this grid's end has to mean that one's too: its first CTA waits before it leaves, and takes the word back.
    if (p.behind && threadIdx.x == 32) {
        uint32_t past;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(past) : "l"(p.plan + p.l.past) : "memory");
        *is_last = past;
    }
    __syncthreads();
    const bool ahead = p.behind && *is_last, holds = p.behind && blockIdx.x == 0;
    if (!ahead) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (p.behind) asm volatile("fence.proxy.async.global;" ::: "memory");  // (the pages are read by TMA)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto leave = [&]() {
        if (!holds) return;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        p.plan[p.l.past] = 0;
    };
    const uint32_t b = blockIdx.x;
    const PagedStart at = paged_load_start(p.plan + p.l.start_small + b * (sizeof(PagedStart) / 4));
    if (at.stamp != p.stamp && threadIdx.x == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_PLAN);
    const uint32_t units = at.units, ctas = at.ctas, u0 = at.u0, u1 = at.u1;
    if (at.stamp != p.stamp || u0 == u1) {
        leave();
        return;
    }
    Walk w;
    w.r = at.r, w.head = at.head, w.tile = at.tile, w.q0 = at.q0, w.n = at.n, w.kv = at.kv;
    w.tiles = paged_tiles(s, w.n, ROWS);
    load_tile(p, w);
    uint32_t step = at.place;  // of the tile
    bool healthy = true;

    if (warp == WARPS) {
        // ---------------- producer: lane i copies one part of a page, half of the keys or values
        const uint32_t box = s.page < KEYS ? s.page : KEYS, boxes = KEYS / box;  // rows of a copy, copies of a step
        const uint32_t mine = lane % (boxes * C::HALVES), which = lane / (boxes * C::HALVES);  // 0: keys, 1: values
        const uint32_t half = mine / boxes, part = mine % boxes;
        const bool copies = which < 2;
        const int outside = (int)(s.pages * s.hkv * s.page);  // a row behind the cache: such a copy is filled with zeros
        uint32_t stage = 0, ph = 1;
        bool bad = false;
        for (uint32_t u = u0; u < u1; u++) {
            const uint32_t key = (w.t.first + step) * KEYS + part * box, block = key / s.page;
            int row = outside;
            if (copies && key < w.t.hi) {
                const int32_t page = p.table[(size_t)w.r * s.max_blocks + block];
                if (page >= 0 && (uint32_t)page < s.pages) row = (int)(((uint32_t)page * s.hkv + w.head) * s.page + key % s.page);
                else if ((block + 1) * s.page > paged_lo(s, paged_hi(s, w.n, w.kv, w.tile * ROWS / s.g))) bad = true;
            }
            if (++step == w.t.steps && u + 1 < u1) {
                step = 0;
                next_tile(p, w);
            }
            if (healthy) healthy = __all_sync(0xffffffffu, mbar_wait(empty + stage, ph, SPIN_LIMIT));
            if (!healthy) break;
            if (lane == 0) mbar_expect_tx(full + stage, C::STAGE);
            __syncwarp();
            uint8_t *to = smem + stage * C::STAGE + (which * C::HALVES + half) * C::PART + part * box * 128;
            if (copies) tma_load_2d(to, which ? &map_v : &map_k, 64 * (int)half, row, full + stage);
            if (++stage == C::STAGES) stage = 0, ph ^= 1;
        }
        if (bad && p.status) atomicOr(p.status, (int)PAGED_STATUS_INDEX);
        // the copies in flight have to land before the CTA leaves
        for (uint32_t i = 0; i < C::STAGES; i++) mbar_wait(full + i, i < stage ? ph ^ 1 : ph, SPIN_LIMIT);
        if (!healthy && lane == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_WAIT);
        leave();
        return;
    }

    // ---------------- four warps, 16 keys of each step
    const uint32_t quad = lane >> 2, pair = 2 * (lane & 3);
    const float c = s.scale * 1.4426950408889634f;  // exponentials to base 2
    const bool q2 = ((uintptr_t)p.q & 3) == 0 && ((p.qv.off | p.qv.head | p.qv.token) & 1) == 0;
    const bool out4 = ((uintptr_t)p.out & 7) == 0 && ((p.ov.off | p.ov.head | p.ov.token) & 3) == 0;
    const uint32_t tid = threadIdx.x;
    // ldmatrix: lane i gives row (i & 7) of matrix i / 8; keys: matrices (keys 0-7, 8-15) of two chunks of 8 elements; values the same, transposed
    const uint32_t k_row = warp * 16 + (lane & 7) + ((lane >> 4) << 3), k_chunk = (lane >> 3) & 1;
    const uint32_t v_row = warp * 16 + (lane & 15), v_chunk = lane >> 4;
    uint32_t stage = 0, ph = 0;
    uint32_t u = u0;
    while (u < u1) {
        const uint32_t steps = min(w.t.steps - step, u1 - u);  // of this tile in this span
        // rows and what they see
        uint32_t lo[2], hi[2];
        uint32_t aq[DP / 16][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t row = w.tile * ROWS + quad + 8 * h, token = row / s.g;
            const bool real = token < w.n;
            hi[h] = real ? paged_hi(s, w.n, w.kv, token) : 0u;
            lo[h] = paged_lo(s, hi[h]);
            const unsigned short *q = (const unsigned short *)p.q + p.qv.off + (uint64_t)(w.q0 + token) * p.qv.token + (uint64_t)(w.head * s.g + row % s.g) * p.qv.head;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t col = 16 * ks + 8 * j + pair;
                    uint32_t x = 0;
                    if (real && col < s.d) x = q2 ? *(const uint32_t *)(q + col) : (uint32_t)q[col] | ((uint32_t)q[col + 1] << 16);
                    aq[ks][2 * j + h] = x;
                }
        }
        const uint32_t tile_lo = paged_lo(s, paged_hi(s, w.n, w.kv, w.tile * ROWS / s.g));
        float o[DP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < DP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        for (uint32_t i = 0; i < steps; i++) {
            if (healthy) healthy = __all_sync(0xffffffffu, mbar_wait(full + stage, ph, SPIN_LIMIT));
            if (!healthy) break;
            const uint32_t kb = s32(smem + stage * C::STAGE), vb = kb + C::HALVES * C::PART;
            float sc[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ks++) {
                uint32_t f[4];
                ldmatrix4<false>(f, kb + (ks / 4) * C::PART + k_row * 128 + (((2 * (ks & 3) + k_chunk) ^ (k_row & 7)) << 4));
                mma16816<BF16>(sc[0], aq[ks], f[0], f[1]);
                mma16816<BF16>(sc[1], aq[ks], f[2], f[3]);
            }
            const uint32_t key0 = (w.t.first + step + i) * KEYS + warp * 16;
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t key = key0 + 8 * t + pair + (e & 1);
                    sc[t][e] = key >= lo[e >> 1] && key < hi[e >> 1] ? sc[t][e] * c : -INFINITY;
                    top[e >> 1] = fmaxf(top[e >> 1], sc[t][e]);
                }
            float base[2], keep[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const float mn = fmaxf(m[h], top[h]);
                base[h] = mn == -INFINITY ? 0.0f : mn;
                keep[h] = exp2_fast(m[h] - base[h]);
                if (mn == m[h]) keep[h] = 1.0f;
                m[h] = mn;
                l[h] *= keep[h];
            }
            if (__any_sync(0xffffffffu, keep[0] != 1.0f || keep[1] != 1.0f)) {
#pragma unroll
                for (int n = 0; n < DP / 8; n++) o[n][0] *= keep[0], o[n][1] *= keep[0], o[n][2] *= keep[1], o[n][3] *= keep[1];
            }
            uint32_t ap[4];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float x = exp2_fast(sc[t][2 * h] - base[h]), y = exp2_fast(sc[t][2 * h + 1] - base[h]);
                    l[h] += x + y;
                    ap[2 * t + h] = pack<BF16>(x, y);
                }
            // values of keys outside the tile's are whatever the page holds: 0 times that must be 0
            uint32_t keep_v[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t key = key0 + 8 * t + pair;
                keep_v[t] = (key >= tile_lo && key < w.t.hi ? 0xffffu : 0u) | (key + 1 >= tile_lo && key + 1 < w.t.hi ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int n = 0; n < DP / 16; n++) {
                uint32_t f[4];
                ldmatrix4<true>(f, vb + (n / 4) * C::PART + v_row * 128 + (((2 * (n & 3) + v_chunk) ^ (v_row & 7)) << 4));
                mma16816<BF16>(o[2 * n], ap, f[0] & keep_v[0], f[1] & keep_v[1]);
                mma16816<BF16>(o[2 * n + 1], ap, f[2] & keep_v[0], f[3] & keep_v[1]);
            }
            // (behind the products: a load may be carried out late, and would read what the next copy brings)
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + stage);
            if (++stage == C::STAGES) stage = 0, ph ^= 1;
        }
        // ---- the four warps' results meet
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
        if ((lane & 3) == 0) {
#pragma unroll
            for (int h = 0; h < 2; h++) meet_m[warp * ROWS + quad + 8 * h] = m[h], meet_l[warp * ROWS + quad + 8 * h] = l[h];
        }
        warps_sync();
        const bool whole = step == 0 && steps == w.t.steps;
        const uint32_t i0 = u - step, i1 = i0 + w.t.steps;  // the tile's place in the sequence
        const uint32_t pf = ROWS * (DP + 2), rows = min(w.n * s.g - w.tile * ROWS, (uint32_t)ROWS);  // (rows that there are)
        float *part = (float *)((uint8_t *)p.plan + p.l.part_small), *mine = part + (size_t)(2 * b + (i0 < u0 ? 0 : 1)) * pf;
        // NR rows of C columns at a time, a thread has four columns of one row: with four rows all columns at once
        auto meeting = [&](auto count) {
            constexpr int NR = decltype(count)::value, C = 512 / NR < DP ? 512 / NR : DP, PITCH = C + 8;
            static_assert(WARPS * NR * PITCH <= MEET, "shared memory");
            const uint32_t row = tid / (C / 4), col = 4 * (tid % (C / 4)), pr = w.tile * ROWS + row, token = pr / s.g, head = w.head * s.g + (pr - token * s.g);
            const bool real = row < rows;
            float f[WARPS], big = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < WARPS; k++) big = fmaxf(big, meet_m[k * ROWS + row % ROWS]);
            const float base = big == -INFINITY ? 0.0f : big;
#pragma unroll
            for (int k = 0; k < WARPS; k++) {
                f[k] = exp2_fast(meet_m[k * ROWS + row % ROWS] - base);
                sum = fmaf(meet_l[k * ROWS + row % ROWS], f[k], sum);
            }
            unsigned short *orow = (unsigned short *)p.out + p.ov.off + (uint64_t)(w.q0 + token) * p.ov.token + (uint64_t)head * p.ov.head;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int c0 = 0; c0 < DP; c0 += C) {
#pragma unroll
                for (int n = 0; n < C / 8; n++)
#pragma unroll
                    for (int h = 0; h < (NR > 8 ? 2 : 1); h++)
                        if (NR >= 8 || quad < NR)
                            *(float2 *)(meet + (warp * NR + quad + 8 * h) * PITCH + 8 * n + pair) = make_float2(o[c0 / 8 + n][2 * h], o[c0 / 8 + n][2 * h + 1]);
                warps_sync();
                if (real) {
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int k = 0; k < WARPS; k++) {
                        const float4 x = *(const float4 *)(meet + (k * NR + row) * PITCH + col);
                        v = make_float4(fmaf(x.x, f[k], v.x), fmaf(x.y, f[k], v.y), fmaf(x.z, f[k], v.z), fmaf(x.w, f[k], v.w));
                    }
                    if (!whole) *(float4 *)(mine + row * DP + c0 + col) = v;
                    else store_half4(orow, c0 + col, s.d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), BF16, out4);
                }
                warps_sync();
            }
            if (real && col == 0) {
                if (!whole) mine[ROWS * DP + row] = big, mine[ROWS * (DP + 1) + row] = sum;
                else if (p.lse) p.lse[(size_t)(w.q0 + token) * s.hq + head] = sum == 0.0f ? -INFINITY : (big + log2f(sum)) * 0.6931471805599453f;
            }
        };
        if (rows <= 4) meeting(std::integral_constant<int, 4>());
        else if (rows <= 8) meeting(std::integral_constant<int, 8>());
        else meeting(std::integral_constant<int, 16>());
        if (!whole) {
            const uint32_t first = paged_holder(units, ctas, i0), last = paged_holder(units, ctas, i1 - 1);
            warps_sync();
            if (tid == 0) {
                uint32_t *count = p.plan + p.l.count_small + first, before;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
                const bool end = before == last - first;
                if (end) *count = 0;  // for the next launch
                *is_last = end;
            }
            warps_sync();
            if (*is_last) {
                // (a tile's first piece is the end of its CTA's span, the others are the beginning of theirs)
                auto piece = [&](uint32_t k) -> const float * { return part + (size_t)(2 * k + (k == first ? 1 : 0)) * pf; };
                const uint32_t quads = min(w.n * s.g - w.tile * ROWS, (uint32_t)ROWS) * (DP / 4);  // four columns of one of the rows that there are
                // a thread has N of them, and B pieces of each in flight: what this takes is the way to memory, and with few rows once
                auto join = [&](auto count, auto batch) {
                    constexpr int N = decltype(count)::value, B = decltype(batch)::value;
                    float rm[N], rl[N];
                    float4 v[N];
#pragma unroll
                    for (int i = 0; i < N; i++) rm[i] = -INFINITY, rl[i] = 0.0f, v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (uint32_t k0 = first; k0 <= last; k0 += B) {
                        float mk[B][N], lk[B][N];
                        float4 x[B][N];
#pragma unroll
                        for (int k = 0; k < B; k++)
#pragma unroll
                            for (int i = 0; i < N; i++) {
                                const uint32_t q = tid + 32 * WARPS * i;
                                const bool there = k0 + k <= last && q < quads;
                                const float *src = piece(there ? k0 + k : first);
                                mk[k][i] = there ? __ldcg(src + ROWS * DP + q / (DP / 4)) : -INFINITY;
                                lk[k][i] = there ? __ldcg(src + ROWS * (DP + 1) + q / (DP / 4)) : 0.0f;
                                x[k][i] = there ? __ldcg((const float4 *)src + q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            }
#pragma unroll
                        for (int i = 0; i < N; i++) {
                            float mm = rm[i];
#pragma unroll
                            for (int k = 0; k < B; k++) mm = fmaxf(mm, mk[k][i]);
                            const float mb = mm == -INFINITY ? 0.0f : mm, keep = exp2_fast(rm[i] - mb);
                            rm[i] = mm;
                            rl[i] *= keep;
                            v[i] = make_float4(v[i].x * keep, v[i].y * keep, v[i].z * keep, v[i].w * keep);
#pragma unroll
                            for (int k = 0; k < B; k++) {
                                const float e = exp2_fast(mk[k][i] - mb);
                                rl[i] = fmaf(lk[k][i], e, rl[i]);
                                v[i] = make_float4(fmaf(x[k][i].x, e, v[i].x), fmaf(x[k][i].y, e, v[i].y), fmaf(x[k][i].z, e, v[i].z), fmaf(x[k][i].w, e, v[i].w));
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const uint32_t q = tid + 32 * WARPS * i;
                        if (q >= quads) break;
                        const uint32_t pr = w.tile * ROWS + q / (DP / 4), tok = pr / s.g, col = 4 * (q % (DP / 4)), head = w.head * s.g + (pr - tok * s.g);
                        unsigned short *to = (unsigned short *)p.out + p.ov.off + (uint64_t)(w.q0 + tok) * p.ov.token + (uint64_t)head * p.ov.head;
                        const float r = rl[i] == 0.0f ? 0.0f : 1.0f / rl[i];
                        store_half4(to, col, s.d, make_float4(v[i].x * r, v[i].y * r, v[i].z * r, v[i].w * r), BF16, out4);
                        if (p.lse && col == 0) p.lse[(size_t)(w.q0 + tok) * s.hq + head] = rl[i] == 0.0f ? -INFINITY : (rm[i] + log2f(rl[i])) * 0.6931471805599453f;
                    }
                };
                if (quads <= 32 * WARPS) join(std::integral_constant<int, 1>(), std::integral_constant<int, 16>());
                else join(std::integral_constant<int, DP / CHUNK>(), std::integral_constant<int, 4>());
            }
        }
        u += steps;
        step = 0;
        if (u < u1) next_tile(p, w);
    }
    if (!healthy && lane == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_WAIT);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

}  // namespace pa

static pa::EncodeTiledFn encode_fn() {
    static const pa::EncodeTiledFn fn = [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (pa::EncodeTiledFn)ptr : nullptr;
    }();
    return fn;
}
static bool encode(const PagedShape &s, const void *base, uint32_t rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box, CUtensorMap &map) {
    const cuuint32_t ones[3] = {1, 1, 1};
    const pa::EncodeTiledFn fn = encode_fn();
    return fn && fn(&map, s.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, (void *)base, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A cache as a matrix [pages * heads * page][d]; boxes of 64 elements (those behind d are filled with zeros) by `rows` rows.
bool paged_cache_map(const PagedShape &s, const void *cache, uint32_t rows, CUtensorMap &map) {
    const cuuint64_t dims[2] = {s.d, (cuuint64_t)s.pages * s.hkv * s.page}, strides[1] = {(cuuint64_t)s.d * 2};
    const cuuint32_t box[2] = {64, rows};
    return encode(s, cache, 2, dims, strides, box, map);
}
// q as [tokens][heads][d]; boxes of 64 elements by the heads of a group by the whole tokens that fit 128 rows: a tile's packed rows in their
// order. False where the view does not allow it (starts and strides of 16 bytes).
bool paged_q_map(const PagedAttnArgs &a, CUtensorMap &map) {
    const PagedShape &s = a.s;
    const char *base = (const char *)a.q + a.qv.off * 2;
    const uint64_t most = 1ull << 40, head = s.hq > 1 ? a.qv.head * 2 : s.d * 2, token = s.tokens > 1 ? a.qv.token * 2 : s.hq * head;
    if (((uintptr_t)base & 15) || head % 16 || token % 16 || head == 0 || token == 0 || head >= most || token >= most || s.tt == 0) return false;
    const cuuint64_t dims[3] = {s.d, s.hq, s.tokens}, strides[2] = {head, token};
    const cuuint32_t box[3] = {64, s.g, s.tt};
    return encode(s, base, 3, dims, strides, box, map);
}

uint32_t paged_attn_small_ctas(int sm_count) { return 2 * (uint32_t)sm_count; }

template <int DP, bool BF16> static cudaError_t small_launch(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, int sm_count, bool pdl, cudaStream_t stream) {
    auto *kernel = pa::paged_attn_small_kernel<DP, BF16>;
    constexpr int SMEM = pa::Cfg<DP>::SMEM;
    static std::once_flag once[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::call_once(once[dev & 63], [&] { e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(paged_attn_small_ctas(sm_count));
    cfg.blockDim = dim3(pa::THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, mk, mv, a);
}

cudaError_t launch_paged_attn_small(const PagedAttnArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    CUtensorMap mk, mv;
    const uint32_t rows = a.s.page < PAGED_SMALL_KEYS ? a.s.page : PAGED_SMALL_KEYS;
    if (!paged_cache_map(a.s, a.k_cache, rows, mk) || !paged_cache_map(a.s, a.v_cache, rows, mv)) return cudaErrorInvalidValue;
    if (a.s.d > 64) return a.s.bf16 ? small_launch<128, true>(a, mk, mv, sm_count, pdl, stream) : small_launch<128, false>(a, mk, mv, sm_count, pdl, stream);
    return a.s.bf16 ? small_launch<64, true>(a, mk, mv, sm_count, pdl, stream) : small_launch<64, false>(a, mk, mv, sm_count, pdl, stream);
}

}  // namespace lb
