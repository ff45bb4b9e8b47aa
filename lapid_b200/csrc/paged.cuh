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

constexpr uint32_t PAGED_STATUS_INDEX = 512, PAGED_STATUS_PAGES = 1024, PAGED_STATUS_WAIT = 2048, PAGED_STATUS_LENGTHS = 4096, PAGED_STATUS_PLAN = 8192;

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

// The tile of a request's new tokens [t0, t1]: at least one step, so that rows without keys are written too
__host__ __device__ inline PagedTile paged_tile_of(const PagedShape &s, uint32_t n, uint32_t kv, uint32_t t0, uint32_t t1, uint32_t keys) {
    PagedTile t;
    t.hi = paged_hi(s, n, kv, t1);
    t.first = paged_lo(s, paged_hi(s, n, kv, t0)) / keys;
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
// Requests of few rows go to one kernel, the others to the other
__host__ __device__ inline bool paged_is_small(const PagedShape &s, uint32_t n) { return n * s.g <= PAGED_SMALL_LIMIT || s.tt == 0; }
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
