// Attention over the pages for requests of many rows: whole prompts and chunks of them, on the 5th-generation tensor cores.
//
//   S = Q K^T;  m = max(scale S), P = exp(scale S - m), l = sum P;  O = sum over the steps of P V;  out = O / l
//
// in one pass over the keys a request's rows may see. A CTA holds two tiles of up to 128 packed rows (token, query head of the group), each with
// its scores S (f32), its weights P (16 bits) and its accumulator O (f32) in tensor memory, so that one tile's products run while the other's
// exponentials are formed. A step is 80 keys (head_dim above 64; else 96): then S, P and O of both tiles fit the 512 columns beside each other,
// and the next step's scores are formed while this one's weights still are. (128 keys with P in S's columns: the next scores wait for the weights' product;
// a step of 128 keys took 3850 cycles, of which the products are 2048.)
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread is a row. S comes from tensor memory into registers, P goes back: the A operand of the second
//              product may lie there. The weights are
//              taken relative to the last maximum that was looked up, and the maximum of the new scores is formed beside them: only where one
//              is more than 2^8 times larger are the weights formed again and O and l rescaled (until then the weights are at most 2^8 and
//              nothing is lost; l and O carry the same factor). Some exponentials are polynomials: see exp2_poly.
//   warps 8, 9 issue `tcgen05.mma` for tile 0, 1: S = Q K^T (both from shared memory) and O += P V (V as it lies in the pages: its rows are
//              the keys, so the descriptor takes it as the transposed operand). A wait costs such a warp, which the softmax leaves few issue slots, 100 cycles and more
//              also when it is over at once: a step has three. (One warp for both tiles spent more time between the products than in them.)
//   warp 10    copies the pages' keys into a ring by TMA
//   warp 11    copies the values, and the next tiles' rows of Q: one box of whole tokens by TMA, or 16 bytes (2, where they are not aligned) a thread
// An event a step ties softmax and products: the scores of the step have been read and the weights of the one before are there. With it the products
// form the next scores, then multiply the weights; the softmax goes on to its exponentials.
// The steps of all requests, heads and tiles are one sequence cut into equal spans, one a CTA (paged.cuh): causal tiles of any length keep every SM
// busy, few rows over many keys spread over all. A tile that a span's end cuts is left in the plan buffer by its CTAs but, as a rule, the one whose span
// ends with the first piece: that one adds the others to its accumulator. Where they are not there yet, or are many, the CTA that comes last adds
// all of them up, in the order of the keys either way and with the same roundings.
//
// What bounds it: a softmax warp's own chain, two warps a scheduler. Heads of 64: a step of 96 keys takes 2050 to 2400 cycles: exponentials 1345 (the special-function unit 47 % busy over
// the kernel), loads, stores and two waits 540, the more of it hidden the further the two tiles are apart; products 26 % of the time. Heads of 128: a step of 80 keys takes some 1720, of which
// both tiles' products are 1280 and their exponentials 1120; over four prompts the tensor pipe is busy 59 % of the time, the special-function unit 52 %. From tile to tile some 6300 cycles pass (heads of 64: 4600), for
// the last product, the rows' stores and the walk; a cut tile's later piece costs 9000, its first 8000 behind the span. Long work runs into the power limit: 512 tokens over
// 32768 keys, 64 query and 8 key heads of 128, 546 to 580 us (0.94 to 1.0 PFLOP/s, the clock at 1.2 to 1.4 GHz); four prompts of up to 4096 tokens, 32 query heads, 306 to 392 us as their lengths fall (0.91 PFLOP/s; when they see all keys 1.06);
// one of 2048 45.3 us; three of up to 3001 through a window of 1024 keys, 14 heads of 64, 61 to 64 us.
//
// Every mbarrier wait is bounded: one that gives up sets a bit in the status word, the roles fall through to the end, tensor memory is released.
#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged.cuh"
#include "pipe.cuh"

namespace lb {

bool paged_cache_map(const PagedShape &s, const void *cache, uint32_t rows, CUtensorMap &map);
bool paged_q_map(const PagedAttnArgs &a, CUtensorMap &map);

namespace pt {

using pipe::add2;
using pipe::fma2;
using pipe::mbar_arrive;
using pipe::mbar_expect_tx;
using pipe::mbar_fence_init;
using pipe::mbar_init;
using pipe::pack2;
using pipe::s32;
using pipe::tma_load_2d;
using pipe::unpack2;

constexpr int TILE = 128, ROWS = PAGED_LARGE_ROWS;
constexpr int MMA_WARP = 8, K_WARP = 10, V_WARP = 11, THREADS = 384;
constexpr int Q_HALF = TILE * 128;  // bytes of 128 rows of 64 elements
// Registers: 384 x 168 at launch = 256 x 208 + 128 x 88
constexpr int REGS_SOFTMAX = 208, REGS_OTHER = 88;
constexpr float LAZY = 8.0f;
constexpr int POLY = 1;  // pairs of every eight whose exponentials are polynomials (with 0, 1, 2 prompts through a window 63.8, 61.5, 66.3 us, 512 tokens over 32768 keys 584, 553, 583)
constexpr uint32_t WAIT_NS = 8000, SPIN_LIMIT = 1u << 18;  // a wait gives up after at most 2.1 seconds

template <int DP> struct Cfg {
    static constexpr int HALVES = DP / 64;
    static constexpr int KEYS = DP > 64 ? 80 : 96;             // PagedShape::large_keys
    static constexpr int HALF = KEYS * 128;                    // bytes of 64 elements of a step's keys (or values)
    static constexpr int STAGE = HALVES * HALF;
    static constexpr int Q_BYTES = 2 * HALVES * Q_HALF;
    static constexpr int STAGES = (224 * 1024 - Q_BYTES) / (2 * STAGE);  // of keys, and as many of values
    static constexpr int SMEM = Q_BYTES + 2 * STAGES * STAGE + 512 + 1024;
    // tensor memory: O of tile t at DP t, S at T_COL + T_STEP t, P behind it
    static constexpr int T_COL = 2 * DP, T_STEP = (512 - T_COL) / 2;
    static_assert(KEYS + KEYS / 2 <= T_STEP && KEYS % 16 == 0, "tensor memory");
};

// Bounded wait. What is waited for is there already, more often than not: the first attempt has no time to sleep (44 cycles, with one 69).
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(s32(bar)), "r"(parity) : "memory");
    for (uint32_t spin = 0; !ok && spin < SPIN_LIMIT; spin++)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(s32(bar)), "r"(parity), "r"(WAIT_NS)
                     : "memory");
    return ok;
}
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }
// Whether the phase is over now
__device__ __forceinline__ bool warp_test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(s32(bar)), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// Operands in shared memory, 128-byte swizzle. K-major: rows of 128 bytes, 8-row groups 1024 bytes apart. Transposed (rows are the K dimension): 8-row
// groups 1024 bytes apart, the next 64 elements of a row `half` bytes further.
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_t(uint32_t saddr, uint32_t half) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(half >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t *r, uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
          "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
          "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
        "%30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
        "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t *r, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
        "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}
// The 80 or 96 columns of a step's scores; 40 or 48 columns of weights
template <int N> __device__ __forceinline__ void load_scores(uint32_t (&x)[N], uint32_t addr) {
#pragma unroll
    for (int i = 0; i + 32 <= N; i += 32) tmem_ld32(x + i, addr + i);
    if constexpr (N % 32 == 16) tmem_ld16(x + N - 16, addr + N - 16);
}
template <int N> __device__ __forceinline__ void store_weights(uint32_t addr, const uint32_t (&w)[N]) {
    tmem_st32(addr, w);
    if constexpr (N % 32 == 16) tmem_st16(addr + 32, w + 32);
    if constexpr (N % 32 == 8) tmem_st8(addr + 32, w + 32);
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

// Behind a wait for loads from tensor memory: nothing may use the registers before it.
template <int N> __device__ __forceinline__ void loaded(uint32_t (&x)[N]) {
    ld_wait();
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(x[i]));
}
// max.NaN: a NaN among the scores stays
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of a pair by Cody and Waite's reduction, x = n + f with |f| <= 1/2, and a polynomial in f, n added to the exponent. The polynomial is 1 at f = 0 and
// otherwise the minimax one (by linear programming; relative error 2.9e-6 at degree 4, at degree 3 7.5e-5, which the weights' type would hide but not the logarithm of their sum). For
// x <= 100. What is below -127, the scores that a mask leaves out among them, is taken as -127: n = -127 takes the 1's exponent to nothing, so the weight is +0 without a test
// (with two tests and selects a pair: window 65.0 instead of 63.6 us). The special-function unit forms 16 exponentials a cycle on an SM, and 128 x 128 of
// them take as long as the two products of 128 x 128 x 128: what it is relieved of here costs five issue slots an element that the schedulers have.
__device__ __forceinline__ void exp2_poly(uint64_t x, float &r0, float &r1) {
    float a, b;
    unpack2(x, a, b);
    x = pack2(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
    const uint64_t t = add2(x, pack2(12582912.0f, 12582912.0f));  // 1.5 2^23: n in the low bits
    const uint64_t f = fma2(add2(t, pack2(-12582912.0f, -12582912.0f)), pack2(-1.0f, -1.0f), x);
    uint64_t y = fma2(f, pack2(0.00958285294f, 0.00958285294f), pack2(0.0559064262f, 0.0559064262f));
    y = fma2(f, y, pack2(0.240240991f, 0.240240991f));
    y = fma2(f, y, pack2(0.693124175f, 0.693124175f));
    y = fma2(f, y, pack2(1.0f, 1.0f));
    float y0, y1, t0, t1;
    unpack2(y, y0, y1);
    unpack2(t, t0, t1);
    r0 = __uint_as_float(__float_as_uint(y0) + (__float_as_uint(t0) << 23));
    r1 = __uint_as_float(__float_as_uint(y1) + (__float_as_uint(t1) << 23));
}
// The weights of N scores, their sums (added to l) and the largest score.
template <bool BF16, int N> __device__ __forceinline__ float weights(const uint32_t (&x)[N], uint64_t c2, uint64_t b2, uint32_t (&w)[N / 2], uint64_t &l0, uint64_t &l1) {
    float top[4];
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const float x0 = __uint_as_float(x[2 * i]), x1 = __uint_as_float(x[2 * i + 1]);
        if (i < 4) asm("max.NaN.f32 %0, %1, %2;" : "=f"(top[i]) : "f"(x0), "f"(x1));
        else top[i & 3] = max3(top[i & 3], x0, x1);
        const uint64_t y = fma2(pack2(x0, x1), c2, b2);
        float e0, e1;
        if ((i & 7) < POLY) {
            exp2_poly(y, e0, e1);
        } else {
            unpack2(y, e0, e1);
            e0 = exp2_fast(e0), e1 = exp2_fast(e1);
        }
        if (i & 1) l1 = add2(l1, pack2(e0, e1));
        else l0 = add2(l0, pack2(e0, e1));
        w[i] = pack<BF16>(e0, e1);
    }
    return max3(max3(top[0], top[1], top[2]), top[3], top[3]);
}

// The same value in all lanes, and the compiler knows it: what the tensor instructions take then stays in uniform registers (a step of 80 keys took
// 2055 cycles without, 1716 with).
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }

struct Walk {
    uint32_t r, head, tile, tiles, n, kv, q0;
    PagedTile t;
    uint32_t i0, u1;         // units: where the tile begins, where the span ends
    uint32_t step, steps;    // first step of the tile here, and how many
    bool two;                // the second tile of 128 has rows
};
// (512 tokens beside 11 single ones take 52.4 us so, 54.5 with the number of tokens in the plan in place of their end: the compiler orders the ends of tiles otherwise. 16 requests of
// eight tokens over 3000 keys 46.3, word by word 46.8.)
__device__ __forceinline__ void load_request(const PagedAttnArgs &p, Walk &w) {
    const uint4 x = ((const uint4 *)(p.plan + p.l.request))[w.r];
    w.q0 = uniform(x.x), w.n = uniform(x.y) - w.q0, w.kv = uniform(x.z);
    w.tiles = paged_tiles(p.s, w.n, paged_large_rows(p.s));
}
// (steps 0: the span ends in what the tile counts in front of its steps)
template <int KEYS> __device__ __forceinline__ bool load_tile(const PagedAttnArgs &p, Walk &w) {
    const uint32_t token0 = 2 * w.tile * p.s.tt;
    w.t = paged_tile_of(p.s, w.n, w.kv, token0, min(token0 + 2 * p.s.tt, w.n) - 1, KEYS);
    w.two = token0 + p.s.tt < w.n;
    const uint32_t begin = w.i0 + PAGED_LARGE_EXTRA, end = w.u1 > begin ? min(w.t.steps, w.u1 - begin) : 0u;
    w.steps = end > w.step ? end - w.step : 0u;
    return w.steps > 0;
}
// The next piece of work of the span; false: none
template <int KEYS> __device__ __forceinline__ bool next_piece(const PagedAttnArgs &p, Walk &w) {
    w.i0 += PAGED_LARGE_EXTRA + w.t.steps;
    if (w.i0 + PAGED_LARGE_EXTRA >= w.u1) return false;
    w.step = 0;
    if (++w.tile == w.tiles) {
        w.tile = 0;
        if (++w.head == p.s.hkv) {
            w.head = 0;
            do {
                w.r++;
                load_request(p, w);
            } while (w.n == 0 || paged_is_small(p.s, w.n));
        }
    }
    return load_tile<KEYS>(p, w);
}
__device__ __forceinline__ uint32_t tile_low(const PagedAttnArgs &p, const Walk &w) { return paged_lo(p.s, paged_hi(p.s, w.n, w.kv, 2 * w.tile * p.s.tt)); }
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(s32(dst)), "l"((uint64_t)map), "r"(x), "r"(y), "r"(z),
                 "r"(s32(bar))
                 : "memory");
}

// 32 columns of a row of out, from `col` on, 32, 16 or 2 bytes at a time. (A store touches the 32 rows of a warp: the wider, the fewer of them.)
template <bool BF16> __device__ __forceinline__ void store32(unsigned short *row, const float *v, uint32_t col, uint32_t d, bool vec, bool wide) {
    if (wide) {
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 16)
            if (col + e < d)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + col + e), "r"(pack<BF16>(v[e], v[e + 1])), "r"(pack<BF16>(v[e + 2], v[e + 3])),
                             "r"(pack<BF16>(v[e + 4], v[e + 5])), "r"(pack<BF16>(v[e + 6], v[e + 7])), "r"(pack<BF16>(v[e + 8], v[e + 9])), "r"(pack<BF16>(v[e + 10], v[e + 11])),
                             "r"(pack<BF16>(v[e + 12], v[e + 13])), "r"(pack<BF16>(v[e + 14], v[e + 15]))
                             : "memory");
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 32; e += 8) {
        if (col + e >= d) break;
        const uint4 y = make_uint4(pack<BF16>(v[e], v[e + 1]), pack<BF16>(v[e + 2], v[e + 3]), pack<BF16>(v[e + 4], v[e + 5]), pack<BF16>(v[e + 6], v[e + 7]));
        if (vec) {
            *(uint4 *)(row + col + e) = y;
        } else {
            const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; i++) row[col + e + 2 * i] = (unsigned short)z[i], row[col + e + 2 * i + 1] = (unsigned short)(z[i] >> 16);
        }
    }
}

// The same for the rows of a warp: four lanes turn their four times 16 bytes round, so that a store has 64 bytes of each of eight rows, and half as many requests leave
// the SM. at[i]: row 4 (lane / 4) + i, or null
template <bool BF16> __device__ __forceinline__ void store32_turned(unsigned short *const (&at)[4], const float *v, uint32_t col, uint32_t d, uint32_t lane) {
    uint32_t y[16];
#pragma unroll
    for (int e = 0; e < 16; e++) y[e] = pack<BF16>(v[2 * e], v[2 * e + 1]);
#pragma unroll
    for (int s = 1; s < 4; s *= 2) {
        const bool up = lane & s;
#pragma unroll
        for (int a = 0; a < 4; a++) {
            if (a & s) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t x = __shfl_xor_sync(0xffffffffu, up ? y[4 * a + e] : y[4 * (a + s) + e], s);
                y[4 * a + e] = up ? x : y[4 * a + e];
                y[4 * (a + s) + e] = up ? y[4 * (a + s) + e] : x;
            }
        }
    }
    col += 8 * (lane & 3);
    if (col >= d) return;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (at[i]) *(uint4 *)(at[i] + col) = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
}

// A cut tile: the CTAs that hold its first and its last step, and whose rows it has
struct Cut {
    uint32_t first, last, q0, n, head, tile;
};
// Adds up the pieces of a tile of 128 rows: piece i of CTA i, [columns / 4][row][4] f32, then the rows' m, then their l (a warp's rows lie behind each
// other). A tile's first piece is the end of its CTA's span, the others are the beginning of theirs. What it takes is the way to memory, so the four warps share
// rows and columns evenly however few rows there are: eight tokens over 8192 keys, 17 pieces of 32 rows a tile, take 19.1 us so, and 41.3 when a thread adds up its own row.
template <int DP, bool BF16> __device__ __forceinline__ void join_pieces(const PagedAttnArgs &p, const Cut &c, uint32_t t, bool vec, bool wide) {
    constexpr uint32_t PF = ROWS * (DP + 2);
    constexpr int B = 4;  // pieces in flight
    const PagedShape &s = p.s;
    const float *const parts = (const float *)((const uint8_t *)p.plan + p.l.part_large);
    const uint32_t first = c.first, last = c.last, lane = threadIdx.x & 31, token0 = (2 * c.tile + t) * s.tt;
    const uint32_t rows = min(s.tt, c.n - token0) * s.g, groups = (rows + 31) / 32;
    auto piece = [&](uint32_t i) -> const float * { return parts + (size_t)(2 * i + (i == first ? 1 : 0)) * PF; };
#pragma unroll 1
    for (uint32_t item = (threadIdx.x >> 5) & 3; item < groups * (DP / 32); item += 4) {
        const uint32_t ch = item / groups, r = 32 * (item - ch * groups) + lane, row = t * TILE + r;
        if (r >= rows) continue;
        float mm = -INFINITY, ll = 0.0f, v[32];
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = 0.0f;
#pragma unroll 1
        for (uint32_t i0 = first; i0 <= last; i0 += B) {
            float m[B], l[B];
            float4 y[B][8];
#pragma unroll
            for (uint32_t k = 0; k < B; k++) {
                const bool there = i0 + k <= last;
                const float *src = piece(there ? i0 + k : last);
                m[k] = there ? __ldcg(src + DP * ROWS + row) : -INFINITY;
                l[k] = there ? __ldcg(src + (DP + 1) * ROWS + row) : 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) y[k][e] = there ? __ldcg((const float4 *)src + (8 * ch + e) * ROWS + row) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            float top = mm;
#pragma unroll
            for (uint32_t k = 0; k < B; k++) top = fmaxf(top, m[k]);
            const float base = top == -INFINITY ? 0.0f : top, keep = exp2_fast(mm - base);
            mm = top;
            ll *= keep;
#pragma unroll
            for (int e = 0; e < 32; e++) v[e] *= keep;
#pragma unroll
            for (uint32_t k = 0; k < B; k++) {
                const float f = exp2_fast(m[k] - base);
                ll = fmaf(l[k], f, ll);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[4 * e] = fmaf(y[k][e].x, f, v[4 * e]);
                    v[4 * e + 1] = fmaf(y[k][e].y, f, v[4 * e + 1]);
                    v[4 * e + 2] = fmaf(y[k][e].z, f, v[4 * e + 2]);
                    v[4 * e + 3] = fmaf(y[k][e].w, f, v[4 * e + 3]);
                }
            }
        }
        const float il = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] *= il;
        const uint32_t local = r / s.g, qh = c.head * s.g + (r - local * s.g);
        const uint64_t at = c.q0 + token0 + local;
        store32<BF16>((unsigned short *)p.out + p.ov.off + at * p.ov.token + (uint64_t)qh * p.ov.head, v, 32 * ch, s.d, vec, wide);
        if (p.lse && ch == 0) p.lse[at * s.hq + qh] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
    }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(THREADS, 1) paged_attn_large_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q, PagedAttnArgs p, bool q_boxes) {
    using C = Cfg<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((0u - s32(smem_raw)) & 1023u);
    uint8_t *k_ring = smem + C::Q_BYTES, *v_ring = k_ring + C::STAGES * C::STAGE;
    uint64_t *k_full = (uint64_t *)(v_ring + C::STAGES * C::STAGE), *k_empty = k_full + C::STAGES, *v_full = k_empty + C::STAGES, *v_empty = v_full + C::STAGES;
    // of each tile: Q in place, read; scores there; scores read and the weights before them there ([event & 1][tile]: the softmax may be at the event behind
    // a piece's last scores before the one in front of it was looked at); product of the weights done; all done
    uint64_t *q_full = v_empty + C::STAGES, *q_empty = q_full + 2, *s_full = q_empty + 2, *ready = s_full + 2, *o_full = ready + 4, *drained = o_full + 2;
    uint32_t *tmem_slot = (uint32_t *)(drained + 2);
    volatile uint32_t *is_last = tmem_slot + 1;
    const PagedShape &s = p.s;
    const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) {
            mbar_init(k_full + i, 1);
            mbar_init(v_full + i, 1);
            mbar_init(k_empty + i, 2);  // both tiles' warps
            mbar_init(v_empty + i, 2);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init(q_full + t, 1);
            mbar_init(q_empty + t, 1);
            mbar_init(s_full + t, 1);
            mbar_init(ready + t, 4);
            mbar_init(ready + 2 + t, 4);
            mbar_init(o_full + t, 1);
            mbar_init(drained + t, 1);
        }
        mbar_fence_init();
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // (the kernel for few rows, started by the next instruction, reads there that what was written in front of this kernel is visible; by a warp that has time)
    if (warp == MMA_WARP + 1) {
        if (lane == 0 && blockIdx.x == 0) asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p.plan + p.l.past), "r"(1u) : "memory");
        __syncwarp();
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    const uint32_t b = blockIdx.x;
    const PagedStart at = paged_load_start(p.plan + p.l.start_large + b * (sizeof(PagedStart) / 4));
    const bool stale = uniform(at.stamp) != p.stamp;
    if (stale && threadIdx.x == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_PLAN);
    const uint32_t units = uniform(at.units), ctas = uniform(at.ctas), u0 = uniform(at.u0), u1 = uniform(at.u1), place = uniform(at.place);
    bool work = !stale && u0 < u1, healthy = true;
    Walk w{};
    if (work) {  // (a span may hold nothing but the front of a tile)
        w.i0 = u0 - place, w.u1 = u1, w.r = uniform(at.r), w.head = uniform(at.head), w.tile = uniform(at.tile), w.q0 = uniform(at.q0), w.n = uniform(at.n), w.kv = uniform(at.kv);
        w.step = place > PAGED_LARGE_EXTRA ? place - PAGED_LARGE_EXTRA : 0u;
        w.tiles = paged_tiles(s, w.n, paged_large_rows(s));
        work = load_tile<C::KEYS>(p, w);
    }

    if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHER));
        if (warp < K_WARP) {
            // ---------------- products of tile t
            // D f32, A and B f16 (0) or bf16 (1); S: both K-major, N = KEYS, A negated for a negative scale; O: B transposed, N = DP
            const uint32_t t = warp - MMA_WARP;
            constexpr uint32_t TYPE = (1u << 4) | ((BF16 ? 1u : 0u) << 7) | ((BF16 ? 1u : 0u) << 10) | ((uint32_t)(TILE >> 4) << 24);
            const uint32_t idesc_s = TYPE | ((uint32_t)(C::KEYS >> 3) << 17) | (s.scale < 0.0f ? 1u << 13 : 0u);
            constexpr uint32_t idesc_o = TYPE | ((uint32_t)(DP >> 3) << 17) | (1u << 16);
            const uint32_t s_col = tmem + C::T_COL + C::T_STEP * t, p_col = s_col + C::KEYS, o_col = tmem + DP * t;
            const uint64_t q_desc = desc_k(s32(smem) + t * C::HALVES * Q_HALF);
            uint32_t ks = 0, kph = 0, vs = 0, vph = 0;  // rings
            uint32_t piece = 0, events = 0;             // pieces of this tile, and times that its softmax was ready
            auto scores = [&](bool last) {
                if (elect_one()) {
                    const uint64_t kd = desc_k(s32(k_ring) + ks * C::STAGE);
#pragma unroll
                    for (int i = 0; i < DP / 16; i++) mma_ss(s_col, q_desc + (i / 4) * (Q_HALF >> 4) + 2 * (i & 3), kd + (i / 4) * (C::HALF >> 4) + 2 * (i & 3), idesc_s, i ? 1u : 0u);
                    commit(s_full + t);
                    commit(k_empty + ks);
                    if (last) commit(q_empty + t);
                }
                __syncwarp();
                if (++ks == C::STAGES) ks = 0, kph ^= 1;
            };
            bool begun = false;  // the piece's first scores are under way
            while (work && healthy) {
                Walk next = w;
                const bool follows = next_piece<C::KEYS>(p, next);
                if (t == 1 && !w.two) {  // the other tile's alone
                    for (uint32_t j = 0; j < w.steps && healthy; j++) {
                        if (!(healthy = warp_wait(k_full + ks, kph) && warp_wait(v_full + vs, vph))) break;
                        if (lane == 0) mbar_arrive(k_empty + ks), mbar_arrive(v_empty + vs);
                        if (++ks == C::STAGES) ks = 0, kph ^= 1;
                        if (++vs == C::STAGES) vs = 0, vph ^= 1;
                    }
                    w = next, work = follows;
                    continue;
                }
                const bool next_mine = follows && (t == 0 || next.two);
                const uint32_t low = tile_low(p, w);
                if (!begun) {
                    if (!(healthy = warp_wait(k_full + ks, kph) && warp_wait(q_full + t, piece & 1))) break;
                    piece++;
                    fence_after();
                    scores(w.steps == 1);
                }
                // Event j: the scores of step j have been read, and the weights of step j - 1 are there. Then the scores behind them may be formed, of step
                // j + 1 or of the next piece's first, and the weights multiplied. (Event `steps`: the last weights are there.) The next piece's Q comes
                // when these scores have read theirs: if it is not there at event `steps` - 1 it is looked for until the last weights are.
                begun = false;
                // the values of step j are there; those of keys that no row of the tile sees are whatever the page holds: 0 times that must be 0 (both warps do it: zeros twice)
                auto values = [&](uint32_t j) -> bool {
                    if (!warp_wait(v_full + vs, vph)) return false;
                    const uint32_t key0 = (w.t.first + w.step + j) * C::KEYS;
                    if (key0 < low || key0 + C::KEYS > w.t.hi) {
                        for (uint32_t i = lane; i < C::KEYS * (DP / 8); i += 32) {
                            const uint32_t key = i / (DP / 8), ch = i % (DP / 8);
                            if (key0 + key < low || key0 + key >= w.t.hi)
                                *(uint4 *)(v_ring + vs * C::STAGE + (ch / 8) * C::HALF + key * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    return true;
                };
                auto multiply = [&](uint32_t j) {
                    if (elect_one()) {
                        const uint64_t vd = desc_t(s32(v_ring) + vs * C::STAGE, C::HALF);
#pragma unroll
                        for (int i = 0; i < C::KEYS / 16; i++) mma_ts(o_col, p_col + 8 * i, vd + i * (2048 >> 4), idesc_o, (j || i) ? 1u : 0u);
                        commit(o_full + t);
                        commit(v_empty + vs);
                    }
                    __syncwarp();
                    if (++vs == C::STAGES) vs = 0, vph ^= 1;
                };
                auto event = [&]() -> bool {
                    if (!warp_wait(ready + 2 * (events & 1) + t, (events >> 1) & 1)) return false;
                    events++;
                    fence_after();
                    return true;
                };
                auto ahead = [&]() {  // the next piece's first scores
                    piece++;
                    begun = true;
                    scores(next.steps == 1);
                };
                for (uint32_t j = 0; j < w.steps; j++) {
                    const bool more = j + 1 < w.steps, first = !more && next_mine && warp_test(k_full + ks, kph) && warp_test(q_full + t, piece & 1);
                    if (!(healthy = (!more || warp_wait(k_full + ks, kph)) && (!j || values(j - 1)) && event())) break;
                    // (the scores first: the softmax waits for them sooner)
                    if (more) scores(j + 2 == w.steps);
                    else if (first) ahead();
                    if (j) multiply(j - 1);
                }
                if (!healthy || !(healthy = values(w.steps - 1))) break;
                // (Q comes some 1200 cycles and more behind its read of the one before, the last weights some 2000: whichever is first)
                if (next_mine)
                    for (uint32_t spin = 0; !begun && spin < SPIN_LIMIT && !warp_test(ready + 2 * (events & 1) + t, (events >> 1) & 1); spin++)
                        if (warp_test(k_full + ks, kph) && warp_test(q_full + t, piece & 1)) ahead();
                if (!(healthy = event())) break;
                multiply(w.steps - 1);
                w = next, work = follows;
            }
            // no product may be under way when tensor memory is released, and nothing may arrive in this CTA's shared memory behind its end
            if (elect_one()) commit(drained + t);
            __syncwarp();
            mbar_wait(drained + t, 0);
            if (!healthy && lane == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_WAIT);
        } else {
            // ---------------- pages: lane i copies one part of a page, half of the keys (warp 10) or values (warp 11)
            const bool values = warp == V_WARP;
            uint8_t *const ring = values ? v_ring : k_ring;
            uint64_t *const full = values ? v_full : k_full, *const empty = values ? v_empty : k_empty;
            const CUtensorMap *const map = values ? &map_v : &map_k;
            constexpr uint32_t box = 16, boxes = C::KEYS / box;  // (rows that every page size and the step are multiples of)
            const bool copies = lane < boxes * C::HALVES;
            const uint32_t half = lane / boxes, part = lane % boxes;
            const int outside = (int)(s.pages * s.hkv * s.page);  // a row behind the cache: such a copy is filled with zeros
            const uint32_t shift = 31 - __clz(s.page);  // (page sizes are powers of two)
            uint32_t st = 0, ph = 1, piece[2] = {0, 0};
            bool bad = false;
            // the rows of Q of a piece, when the scores of the one before have read theirs
            const uint32_t tile_rows = s.tt * s.g;
            const bool vec = ((uintptr_t)p.q & 15) == 0 && ((p.qv.off | p.qv.head | p.qv.token) & 7) == 0;
            auto load_q = [&]() {
                for (int t = 0; t < (w.two ? 2 : 1); t++) {
                    if (piece[t] && !(healthy = warp_wait(q_empty + t, (piece[t] - 1) & 1))) return;
                    piece[t]++;
                    const uint32_t token0 = (2 * w.tile + t) * s.tt;
                    uint8_t *const dst0 = smem + t * C::HALVES * Q_HALF;
                    if (q_boxes) {  // (tokens behind the request's are some other's, or zeros: such rows go nowhere)
                        if (elect_one()) {
                            mbar_expect_tx(q_full + t, C::HALVES * tile_rows * 128);
                            for (int h = 0; h < C::HALVES; h++) tma_load_3d(dst0 + h * Q_HALF, &map_q, 64 * h, (int)(w.head * s.g), (int)(w.q0 + token0), q_full + t);
                        }
                        __syncwarp();
                        continue;
                    }
                    for (uint32_t i = lane; i < tile_rows * (DP / 8); i += 32) {
                        const uint32_t row = i / (DP / 8), ch = i % (DP / 8), local = row / s.g, token = token0 + local;
                        const bool real = token < w.n && 8 * ch < s.d;
                        const unsigned short *src = (const unsigned short *)p.q;
                        if (real) src += p.qv.off + (uint64_t)(w.q0 + token) * p.qv.token + (uint64_t)(w.head * s.g + (row - local * s.g)) * p.qv.head + 8 * ch;
                        uint8_t *dst = dst0 + (ch / 8) * Q_HALF + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
                        if (vec) {
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s32(dst)), "l"(src), "r"(real ? 16u : 0u) : "memory");
                        } else {
                            uint32_t x[4] = {0, 0, 0, 0};
                            if (real)
                                for (int e = 0; e < 4; e++) x[e] = (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16);
                            *(uint4 *)dst = make_uint4(x[0], x[1], x[2], x[3]);
                        }
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(q_full + t);
                }
            };
            while (work && healthy) {
                const uint32_t low = tile_low(p, w);
                auto row_of = [&](uint32_t j) -> int {
                    const uint32_t key = (w.t.first + w.step + j) * C::KEYS + part * box, block = key >> shift;
                    if (!copies || key >= w.t.hi) return outside;
                    const int32_t page = p.table[(size_t)w.r * s.max_blocks + block];
                    if (page >= 0 && (uint32_t)page < s.pages) return (int)(((uint32_t)page * s.hkv + w.head) * s.page + (key & (s.page - 1)));
                    if ((block + 1) * s.page > low) bad = true;
                    return outside;
                };
                int row = row_of(0);
                if (values) load_q();
                for (uint32_t j = 0; j < w.steps && healthy; j++) {
                    const int now = row;
                    if (j + 1 < w.steps) row = row_of(j + 1);
                    if (!(healthy = warp_wait(empty + st, ph))) break;
                    if (lane == 0) mbar_expect_tx(full + st, C::STAGE);
                    __syncwarp();
                    if (copies) tma_load_2d(ring + st * C::STAGE + half * C::HALF + part * box * 128, map, 64 * (int)half, now, full + st);
                    if (++st == C::STAGES) st = 0, ph ^= 1;
                }
                if (healthy) work = next_piece<C::KEYS>(p, w);
            }
            if (bad && p.status) atomicOr(p.status, (int)PAGED_STATUS_INDEX);
            // the copies in flight have to land before the CTA leaves
            for (uint32_t i = 0; i < C::STAGES; i++) mbar_wait(full + i, i < st ? ph ^ 1 : ph);
            if (values)
                for (int t = 0; t < 2; t++)
                    if (piece[t]) mbar_wait(q_full + t, (piece[t] - 1) & 1);
            if (!healthy && lane == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_WAIT);
        }
    } else {
        // ---------------- softmax: tile t, a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
        const uint32_t t = warp >> 2, row = threadIdx.x & 127, lanes = (32 * (warp & 3)) << 16;
        const uint32_t s_col = tmem + C::T_COL + C::T_STEP * t + lanes, p_col = s_col + C::KEYS, o_col = tmem + DP * t + lanes;
        const float c = fabsf(s.scale) * 1.4426950408889634f;  // exponentials to base 2
        const bool vec = ((uintptr_t)p.out & 15) == 0 && ((p.ov.off | p.ov.head | p.ov.token) & 7) == 0, wide = ((uintptr_t)p.out & 31) == 0 && ((p.ov.off | p.ov.head | p.ov.token | s.d) & 15) == 0;
        float *const parts = (float *)((uint8_t *)p.plan + p.l.part_large);
        constexpr uint32_t PF = ROWS * (DP + 2);
        auto tile_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + t) : "memory"); };
        uint32_t k = 0, events = 0;  // steps so far, and times that it was ready
        const uint32_t local = row / s.g, member = row - local * s.g;
        for (; work; work = next_piece<C::KEYS>(p, w)) {
            if (t == 1 && !w.two) continue;
            const uint32_t token = (2 * w.tile + t) * s.tt + local, qh = w.head * s.g + member;
            const bool real = local < s.tt && token < w.n;
            // (rows that are none see everything: their results go nowhere, and they ask for no mask)
            const uint32_t hi = real ? paged_hi(s, w.n, w.kv, token) : ~0u, lo = real ? paged_lo(s, hi) : 0u;
            float m = -INFINITY, base = 0.0f;  // the maximum that the weights refer to
            uint64_t l0 = 0, l1 = 0;           // two pairs of sums
            const uint64_t c2 = pack2(c, c);
            uint32_t x[C::KEYS];
            auto wait_scores = [&](uint32_t step) -> bool {
                if (!warp_wait(s_full + t, step & 1)) return false;
                fence_after();
                return true;
            };
            auto say_ready = [&]() {
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ready + 2 * (events & 1) + t);
                events++;
            };
            if (healthy && (healthy = wait_scores(k))) {
                load_scores(x, s_col);
                loaded(x);
                say_ready();
            }
            for (uint32_t j = 0; j < w.steps && healthy; j++) {
                const uint32_t key0 = (w.t.first + w.step + j) * C::KEYS;
                if (__any_sync(0xffffffffu, (real && key0 + C::KEYS > hi) || key0 < lo)) {
                    // a bit for each column that the row sees
                    const uint32_t from = lo > key0 ? min(lo - key0, (uint32_t)C::KEYS) : 0u, to = hi > key0 ? min(hi - key0, (uint32_t)C::KEYS) : 0u;
#pragma unroll
                    for (uint32_t g = 0; g < (uint32_t)C::KEYS; g += 32) {
                        const uint32_t below = to > g ? (to - g >= 32 ? ~0u : (1u << (to - g)) - 1) : 0u, out = from > g ? (from - g >= 32 ? ~0u : (1u << (from - g)) - 1) : 0u;
                        const uint32_t bits = below & ~out;
#pragma unroll
                        for (uint32_t i = 0; i < 32 && g + i < (uint32_t)C::KEYS; i++)
                            if (!(bits & (1u << i))) x[g + i] = 0xff800000u;
                    }
                }
                if (j == 0) {  // no maximum as yet: the scores' own
                    float a4[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) a4[i] = fmaxf(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
#pragma unroll
                    for (int i = 8; i < C::KEYS; i += 2) a4[(i / 2) & 3] = fmaxf(fmaxf(a4[(i / 2) & 3], __uint_as_float(x[i])), __uint_as_float(x[i + 1]));
                    m = fmaxf(fmaxf(a4[0], a4[1]), fmaxf(a4[2], a4[3])) * c;
                    base = m == -INFINITY ? 0.0f : m;
                }
                uint32_t wt[C::KEYS / 2];
                uint64_t n0 = l0, n1 = l1;
                float top = weights<BF16>(x, c2, pack2(-base, -base), wt, n0, n1);
                const bool sound = top < INFINITY;  // (false for NaN and +inf: such a row is NaN)
                top *= c;
                // the product of the step before is done: P's columns are free, O may change
                if (k > 0 && !(healthy = warp_wait(o_full + t, (k - 1) & 1))) break;
                fence_after();  // (the stores to P's columns and the loads and stores of O come behind that product)
                if (__any_sync(0xffffffffu, real && top > m + LAZY)) {
                    const float mn = fmaxf(m, top), bn = mn == -INFINITY ? 0.0f : mn, keep = exp2_fast(m - bn);
                    m = mn, base = bn;
                    const uint64_t k2 = pack2(keep, keep);
                    n0 = pipe::mul2(l0, k2), n1 = pipe::mul2(l1, k2);
                    if (j) {
#pragma unroll 1
                        for (int i = 0; i < DP / 32; i++) {
                            uint32_t o[32];
                            tmem_ld32(o, o_col + 32 * i);
                            loaded(o);
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st32(o_col + 32 * i, o);
                        }
                    }
                    weights<BF16>(x, c2, pack2(-base, -base), wt, n0, n1);
                }
                l0 = n0, l1 = n1;
                if (!sound) l0 = pack2(NAN, NAN);
                store_weights(p_col, wt);
                k++;
                const bool more = j + 1 < w.steps;
                if (more && !(healthy = wait_scores(k))) break;
                if (more) load_scores(x, s_col);
                st_wait();
                if (more) loaded(x);
                say_ready();
            }
            // ---- the piece is done: O is complete behind its last product
            float a0, a1, a2, a3;
            unpack2(l0, a0, a1);
            unpack2(l1, a2, a3);
            float l = (a0 + a1) + (a2 + a3);
            const bool whole = w.steps == w.t.steps;
            const uint32_t first_unit = w.i0 + PAGED_LARGE_EXTRA;
            // A cut tile's first piece is the end of a span, its others are the beginnings of theirs. When they are there as the first is done they are added here, so that
            // the first need not go through memory. It is worth a look when the second of two is well shorter than the span, and when there are three (of few rows join_pieces is quicker).
            // 2048 tokens 59.1 -> 52.4 us, 512 beside 11 requests' single ones 48.6 -> 45.4.
            const uint32_t first = whole ? b : paged_holder(units, ctas, first_unit), last = whole ? b : paged_holder(units, ctas, first_unit + w.t.steps - 1);
            uint32_t *const count = p.plan + p.l.count_large + 2 * first + t;
            uint32_t others = 0;
            if (b == first && !whole && ((last == first + 2 && (w.n - 2 * w.tile * s.tt) * s.g > 64) || (last == first + 1 && w.t.steps - w.steps + 2 * PAGED_LARGE_EXTRA <= u1 - u0))) {
                if (row == 0) {
                    uint32_t there;
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(count) : "memory");
                    there = there == last - first ? there : 0;
                    if (there) *count = 0;  // for the next launch
                    is_last[t] = there;
                }
                tile_sync();
                others = is_last[t];
                tile_sync();
            }
            if (healthy) healthy = warp_wait(o_full + t, (k - 1) & 1);
            fence_after();
            unsigned short *orow = (unsigned short *)p.out + p.ov.off + (uint64_t)(w.q0 + token) * p.ov.token + (uint64_t)qh * p.ov.head;
            auto store_lse = [&](float mm, float ll) {
                if (p.lse && real) p.lse[(size_t)(w.q0 + token) * s.hq + qh] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
            };
            const uint32_t prow = t * TILE + row;
            float *mine = parts + (size_t)(2 * b + (w.step ? 0 : 1)) * PF;
            const bool here = whole || others;
            const float *const theirs = parts + (size_t)2 * (first + 1) * PF;  // and 2 PF behind it
            float keep = 1.0f, add[2] = {0.0f, 0.0f};
            if (others) {
                const float m1 = __ldcg(theirs + DP * ROWS + prow), m2 = others > 1 ? __ldcg(theirs + (DP + 2 * (DP + 2)) * ROWS + prow) : -INFINITY;
                const float mm = fmaxf(fmaxf(m, m1), m2), mb = mm == -INFINITY ? 0.0f : mm;
                keep = exp2_fast(m - mb), add[0] = exp2_fast(m1 - mb), add[1] = exp2_fast(m2 - mb);
                m = mm;
                l = fmaf(__ldcg(theirs + (DP + 1) * ROWS + prow), add[0], l * keep);
                if (others > 1) l = fmaf(__ldcg(theirs + (DP + 1 + 2 * (DP + 2)) * ROWS + prow), add[1], l);
            }
            const float inv = here ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
            // (2048 tokens 47.1 us, row by row 48.8; four prompts of up to 4096 382 and 393; 16 requests of eight tokens, 32 rows each, 46.3 row by row, 46.8 turned)
            const bool turned = vec && here && (w.n - 2 * w.tile * s.tt) * s.g > 64;
            unsigned short *rows4[4] = {};
            if (turned)
#pragma unroll
                for (int i = 0; i < 4; i++) rows4[i] = (unsigned short *)__shfl_sync(0xffffffffu, real ? (unsigned long long)orow : 0ull, (lane & 28) + i);
#pragma unroll 1
            for (int i = 0; i < DP / 32; i++) {
                uint32_t o[32];
                tmem_ld32(o, o_col + 32 * i);
                loaded(o);
                float v[32];
#pragma unroll
                for (int e = 0; e < 32; e++) v[e] = __uint_as_float(o[e]) * keep;
#pragma unroll 1
                for (uint32_t k = 0; k < others; k++) {
                    const float4 *src = (const float4 *)(theirs + (size_t)k * 2 * PF) + 8 * i * ROWS + prow;
                    const float f = k ? add[1] : add[0];
                    float4 y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = __ldcg(src + e * ROWS);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        v[4 * e] = fmaf(y[e].x, f, v[4 * e]);
                        v[4 * e + 1] = fmaf(y[e].y, f, v[4 * e + 1]);
                        v[4 * e + 2] = fmaf(y[e].z, f, v[4 * e + 2]);
                        v[4 * e + 3] = fmaf(y[e].w, f, v[4 * e + 3]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; e++) v[e] *= inv;
                if (here) {
                    if (turned) store32_turned<BF16>(rows4, v, 32 * i, s.d, lane);
                    else if (real) store32<BF16>(orow, v, 32 * i, s.d, vec, wide);
                } else if (real) {
#pragma unroll
                    for (int e = 0; e < 8; e++) ((float4 *)mine)[(8 * i + e) * ROWS + prow] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                }
            }
            fence_before();
            if (here) {
                store_lse(m, l);
                continue;
            }
            if (real) mine[DP * ROWS + prow] = m, mine[(DP + 1) * ROWS + prow] = l;
            tile_sync();
            if (row == 0) {
                uint32_t before;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
                const bool end = before == last - first;
                if (end) *count = 0;  // for the next launch
                is_last[t] = end;
            }
            tile_sync();
            if (is_last[t]) join_pieces<DP, BF16>(p, Cut{first, last, w.q0, w.n, w.head, w.tile}, t, vec, wide);
            tile_sync();  // (without it the compiler merges this end with the others' and spills 330 bytes in the steps: 640 instead of 580 us for 512 rows over 32768 keys)
        }
        if (!healthy && lane == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_WAIT);
    }
    fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace pt

uint32_t paged_attn_large_ctas(int sm_count) { return (uint32_t)sm_count; }

template <int DP, bool BF16> static cudaError_t large_launch(const PagedAttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, const CUtensorMap &mq, bool boxes, int sm_count, bool pdl, cudaStream_t stream) {
    auto *kernel = pt::paged_attn_large_kernel<DP, BF16>;
    constexpr int SMEM = pt::Cfg<DP>::SMEM;
    static std::once_flag once[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::call_once(once[dev & 63], [&] { e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(paged_attn_large_ctas(sm_count));
    cfg.blockDim = dim3(pt::THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, mk, mv, mq, a, boxes);
}

cudaError_t launch_paged_attn_large(const PagedAttnArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    CUtensorMap mk, mv, mq{};
    constexpr uint32_t rows = 16;
    if (!paged_cache_map(a.s, a.k_cache, rows, mk) || !paged_cache_map(a.s, a.v_cache, rows, mv)) return cudaErrorInvalidValue;
    const bool boxes = paged_q_map(a, mq);
    if (a.s.d > 64) return a.s.bf16 ? large_launch<128, true>(a, mk, mv, mq, boxes, sm_count, pdl, stream) : large_launch<128, false>(a, mk, mv, mq, boxes, sm_count, pdl, stream);
    return a.s.bf16 ? large_launch<64, true>(a, mk, mv, mq, boxes, sm_count, pdl, stream) : large_launch<64, false>(a, mk, mv, mq, boxes, sm_count, pdl, stream);
}

}  // namespace lb
