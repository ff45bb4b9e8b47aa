// Geometry of the attention over a paged cache that the plan (paged.cu) and the attention kernels (paged_attn*.cu) share: what is
// a row, a tile of rows, a unit of work, and where the words of a plan buffer lie.
//
// The query heads of one key/value head read the same keys, so they are rows of one tile: packed row p = token * g + head
// of the group (g = q_heads / kv_heads). A tile is PAGED_SMALL_ROWS consecutive packed rows of one request and one key/value head, or twice the whole
// tokens that fit 128 rows (PagedShape::tt of them); it walks the keys that any of its rows may see in steps of PAGED_SMALL_KEYS or PagedShape::large_keys: the units.
// All units of a launch form one sequence (request, head, tile, step), cut into equal spans, one per CTA, whatever the lengths are.
// A tile cut by the end of a span is added up from its pieces. A tile of many rows counts PAGED_LARGE_EXTRA units more than its steps, in front of them:
// what its beginning and its end cost.
#pragma once
#include <stdint.h>

#include "kernels.h"

namespace lb {

constexpr uint32_t PAGED_STATUS_INDEX = 512, PAGED_STATUS_PAGES = 1024, PAGED_STATUS_WAIT = 2048, PAGED_STATUS_LENGTHS = 4096, PAGED_STATUS_PLAN = 8192, PAGED_STATUS_LOGITS = 16384;

struct PagedTile {
    uint32_t first, steps;  // its steps over the keys: [first, first + steps), in units of `keys`
    uint32_t hi;            // keys of the request that any row may see: below hi
};

// Keys that token `t` (of `n` new ones) of a request with `kv` keys may see: [lo, hi)
__host__ __device__ inline uint32_t paged_hi(const PagedShape &s, uint32_t n, uint32_t kv, uint32_t t) {
    if (s.mask != PAGED_CAUSAL) return kv;
    const uint32_t back = n - 1 - t;  // new tokens behind this one
    return kv > back ? kv - back : 0u;
}
__host__ __device__ inline uint32_t paged_lo(const PagedShape &s, uint32_t hi) { return s.window && hi > s.window ? hi - s.window : 0u; }
// The first key that any token from `t0` on may see. Of a tree: where a token that has no ancestor may begin to look, since the tokens' places say nothing of their depth.
__host__ __device__ inline uint32_t paged_tile_lo(const PagedShape &s, uint32_t n, uint32_t kv, uint32_t t0) { return paged_lo(s, paged_hi(s, n, kv, s.tree ? 0u : t0)); }

// A drafted token's row of the tree buffer: [0] how many ancestors it has, behind it the bits of those and of itself (bit i of word w: token 32 w + i of the request; with a
// window the near ones). Of the cached keys it sees those from `lo` on.
__host__ __device__ inline uint32_t paged_tree_lo(const PagedShape &s, uint32_t cached, uint32_t depth) { return paged_lo(s, cached + depth + 1); }
#ifdef __CUDACC__
// 32 of its bits, from token i0 on (which may lie in front of the first)
__device__ __forceinline__ uint32_t paged_tree_bits(const uint32_t *row, uint32_t words, int32_t i0) {
    const int32_t w = i0 >> 5;
    const uint32_t a = (uint32_t)w < words ? row[1 + w] : 0u, b = (uint32_t)(w + 1) < words ? row[2 + w] : 0u;
    return __funnelshift_r(a, b, (uint32_t)i0 & 31);
}
#endif

// The tile of a request's new tokens [t0, t1]: at least one step, so that rows without keys are written too
__host__ __device__ inline PagedTile paged_tile_of(const PagedShape &s, uint32_t n, uint32_t kv, uint32_t t0, uint32_t t1, uint32_t keys) {
    PagedTile t;
    t.hi = paged_hi(s, n, kv, t1);
    t.first = paged_tile_lo(s, n, kv, t0) / keys;
    const uint32_t end = (t.hi + keys - 1) / keys;
    t.steps = end > t.first ? end - t.first : 1u;
    return t;
}
// Tile i of a request
__host__ __device__ inline PagedTile paged_tile(const PagedShape &s, uint32_t n, uint32_t kv, uint32_t i, uint32_t rows, uint32_t keys) {
    const uint32_t p0 = i * rows, p1 = p0 + rows < n * s.g ? p0 + rows : n * s.g;  // packed rows
    return paged_tile_of(s, n, kv, p0 / s.g, (p1 - 1) / s.g, keys);
}
__host__ __device__ inline uint32_t paged_tiles(const PagedShape &s, uint32_t n, uint32_t rows) { return (n * s.g + rows - 1) / rows; }
// Requests of few rows go to one kernel, the others to the other. Of a tree's step all go to one, by the most tokens a request may have: a launch that finds nothing to do takes
// 2 us. (64 requests over 2048 to 4096 keys, most of them of one token: beside a tree of 16 138.8 us, beside four 142.1, beside one of 64 185.2; the same lengths with the mask CAUSAL, where each request has its kernel, 134.2,
// 143.0 and 134.8. 64 of 2, 4, 8 and 16 tokens 151.5, 152.5, 151.7 and 148.7, CAUSAL 137.9, 162.5, 189.4 and 150.2.)
__host__ __device__ inline bool paged_is_small(const PagedShape &s, uint32_t n) { return (s.tree ? s.max_new * s.g <= PAGED_SMALL_LIMIT_TREE : n * s.g <= PAGED_SMALL_LIMIT) || s.tt == 0; }
// A tree's tiles of more than 32 rows that are cut into many pieces are added up by a kernel of its own (paged_attn_tc.cu); of fewer rows the last CTA of a tile is quicker than a launch (32 rows over 4096
// keys 15.4 and 16.8 us, 64 rows 20.2 and 16.4)
__host__ __device__ inline bool paged_joins_apart(const PagedShape &s) { return s.tree && s.max_new * s.g > 32; }
__host__ __device__ inline uint32_t paged_large_rows(const PagedShape &s) { return 2 * s.tt * s.g; }

// What a CTA of an attention launch begins with (one 64-byte line of the plan, so that one load brings it all); u0 == u1: it has nothing to do
struct alignas(16) PagedStart {
    uint32_t stamp, units, ctas, u0;  // what the plan was made for; the launch's steps and CTAs; this one's span [u0, u1)
    uint32_t u1, r, head, tile;
    uint32_t place, q0, n, kv;        // units of the tile in front of u0; the request's first row of q, new tokens and keys
    uint32_t unused[4];
};
__device__ inline PagedStart paged_load_start(const uint32_t *words) {
    PagedStart x;
    const uint4 *src = (const uint4 *)words;
    *(uint4 *)&x.stamp = src[0];
    *(uint4 *)&x.u1 = src[1];
    *(uint4 *)&x.place = src[2];
    return x;
}

// Span of CTA b of c over u units, and the CTA whose span holds unit x
__host__ __device__ inline uint32_t paged_span(uint32_t u, uint32_t c, uint32_t b) { return (uint32_t)((uint64_t)u * b / c); }
__host__ __device__ inline uint32_t paged_holder(uint32_t u, uint32_t c, uint32_t x) { return (uint32_t)((((uint64_t)x + 1) * c - 1) / u); }

}  // namespace lb
