// Which drafted tokens the model's probabilities accept, and the token behind them.
//
// A request's first token is the text's last; its logits z give the distribution of what follows, P = softmax(z / T) (T = 0: the largest alone). The walk begins there. The
// children of the node v it has reached are tried in their order: with the draft's distribution D of v, child c with token x is accepted when u_c D(x) < P(x), else P becomes what D
// left, max(P - D, 0) / sum of it; without D (candidates that were chosen, not drawn) when u_c < P(x), else x leaves P. An accepted child is the next v; when none is,
// the token behind the path is the first t with P(0) + .. + P(t) > w. Whatever the drafts are, the tokens are then distributed as the model's own.
//
// Decisions are comparisons, so what decides is 64 bits wide. With u = 2^-53 a sum of weights is off by at most 7e-14 of itself (a weight e^-x by (x + 8) u, x at most 15.3 in their mean; at most 530 additions), so a
// result differs from the definition's only where a number drawn is next to a border: within 2e-13 of it; within 1e-10 behind rejected candidates, whose weights are taken off a sum while 2^-10 of it is left; behind
// rejected drafts within 3e-13 over the part of all probability that max(P - D, 0) left (a draft that is the model but for its rounding to 32 bits leaves some 1e-8).
// A node's sum is formed in 32 bits first, which is off by less than SURE of it; a child whose test that leaves open, and what is drawn from, gets it again in 64 bits. (Half of the 64-bit operations that a sum of
// weights for every node would be; an SM does 64 of these a cycle.)
//
// A request belongs to a cluster of CTAs, each with a part of the vocabulary, a warp of it to a warp; only the rows on the path are read. A level is a pass over the node's logits (largest and sum), an
// exchange over the cluster's shared memory, and the children's tests, whose tokens, numbers and values were fetched meanwhile. What decides comes from rank 0's loads and from the exchanged sums
// alone, so that the CTAs of a cluster always take the same way.
//
// What bounds it is the chain of a level, some 7000 cycles (the row and the children's values 1350, weights 1340, sums 620, telling and the barrier 900, reading them 1280, the test 890, going on 450), and at the end 64-bit weights, 25 to 30
// instructions each. By the paths drawn one chain of eight over 128256 tokens takes 24 to 30 us, of which 11 are three levels and 8 the two sums behind a rejection; 16 trees over 32000 20 to 22; 64 trees over 128256 92 to
// 98; 32 greedy ones over 50257 22 to 23. (The figures beside the choices below were taken with a weight's series one power shorter, which is 1.5 % less.)
#include <cuda.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "pipe.cuh"

namespace lb {

namespace pv {

using pipe::s32;

constexpr uint32_t WARPS = 16, THREADS = 32 * WARPS, MOST_CTAS = 16;  // of a cluster

// How far a sum of weights in 32 bits is off, relative: z - top, log2(e), that over T and the product are rounded, 4 2^-24 of the exponent x of e^x, whose mean over the weights is at most ln 2^22 = 15.3 (their
// entropy); a weight is the product of powers of 2, 2^-22 and a product's 2^-24 each, to the thread's largest (as that grows, at most 64 times: PART_MOST), the warp's, the CTA's and the
// cluster's; at most 90 additions, 2^-24 each. In all 3e-5, of which 2^-14 is twice as much. A child's own weight in 32 bits, where its test is decided by it, is 1e-30 or more, so x at most 69.1 and it is off by
// 1.7e-5: both together stay below 2^-14 too.
constexpr double SURE = 0x1p-14;
constexpr uint32_t PART_MOST = 64 * 32 * 16;  // a warp's places

// What the warps of the cluster tell each other comes in two sets: a warp writes a set again only when all have read it, which they say with the exchange between.
struct Shared {
    uint64_t quick[2][MOST_CTAS * WARPS];  // a warp's largest logit and its sum in 32 bits; at temperature 0 the largest logit (as `ordered`) and the complement of its place
    double sum[2][MOST_CTAS * WARPS];      // a warp's sum in 64 bits
    double root[16];                       // 2^(j / 16)
    uint32_t n;                            // of the request
    float temperature;
};
struct Node {  // a drafted token
    int32_t token;
    float accept, logit, draft;  // (the latter two when the walk is at its parent)
};

// value, taken, node and parent of each of `most` tokens, and a bit for each token of the vocabulary's part
constexpr int SMEM_MOST = 160 * 1024;
constexpr size_t shared_bytes(uint32_t most, uint32_t part) { return sizeof(Shared) + most * (2 * sizeof(double) + sizeof(Node) + 4) + (size_t)WARPS * part / 8; }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t of_rank(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(s32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void put(uint32_t at, uint32_t x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }
__device__ __forceinline__ void put(uint32_t at, float x) { put(at, __float_as_uint(x)); }
__device__ __forceinline__ void put(uint32_t at, uint64_t x) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(x) : "memory"); }
__device__ __forceinline__ void put(uint32_t at, double x) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(x) : "memory"); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// (larger, and of equal ones the lower index; NaN stays)
__device__ __forceinline__ void better(float &top, uint32_t &at, float t, uint32_t i) {
    if (t > top || (t == top && i < at)) at = i;
    top = max_nan(top, t);
}

// Weights e^((z - top) / T): with c = 16 log2(e) / T and n the whole number nearest to (z - top) c, 2^(n / 16) from a table of 16 (of which any lanes may read any without a bank
// conflict) and the exponent, times the series of 2^(f / 16), |f| <= 1/2, to the sixth power, which leaves 4.4e-16: thirteen operations of 64 bits. (To the fifth it would leave 1.5e-13, which is seen where a draft that
// is nearly the model leaves 1e-8 of all probability.) A weight below e^-700 is 0, as that of -inf is, whatever T is.
struct Weight {
    const double *root;
    double top, c = 0.0;
    float low;
    __device__ __forceinline__ Weight(const double *table, float t) : root(table), top((double)t), low(t) {}
    __device__ __forceinline__ void set(float temperature) {
        c = 23.083120654223414 / (double)temperature;
        low = fmaxf(__double2float_ru(top - 700.0 * (double)temperature), -3.4028235e38f);  // (rounded up: below e^-708 the exponent has no place)
    }
    __device__ __forceinline__ double operator()(float z) const {
        const double d = (double)z - top, magic = 6755399441055744.0;  // 1.5 2^52
        const double k = fma(d, c, magic), f = fma(d, c, magic - k);
        const int n = __double2loint(k);
        // (ln 2 / 16)^i / i!
        double p = fma(f, 9.181219573844438e-12, 1.271587195055813e-09);
        p = fma(f, p, 1.467610032291943e-07);
        p = fma(f, p, 1.3550807779497455e-05);
        p = fma(f, p, 0.0009383847928089871);
        p = fma(f, p, 0.04332169878499658);
        p = fma(f, p, 1.0);
        p *= root[n & 15];
        p = __hiloint2double(__double2hiint(p) + (n & ~15) * 65536, __double2loint(p));
        return z < low ? 0.0 : p;
    }
};
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// max(x, 0) by the sign bit
__device__ __forceinline__ double positive(double x) {
    const int keep = ~(__double2hiint(x) >> 31);
    return __hiloint2double(__double2hiint(x) & keep, __double2loint(x) & keep);
}
// Whole numbers in the order of the floats, the same one for both zeros (-0.0 + 0.0 is 0.0), NaN on top
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? ~0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// E elements of a row whose tokens are the places [from, from + vocab) behind `row`, which is aligned to 16 bytes, from place `i` (a multiple of E) on; `none` outside
template <int SRC, int E> __device__ __forceinline__ void load_row(float *x, const void *row, uint32_t i, uint32_t from, uint32_t end, float none) {
    if (i >= from && i + E <= end) {
        if constexpr (SRC == ACT_F32) {
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                const float4 v = *(const float4 *)((const float *)row + i + e);
                x[e] = v.x, x[e + 1] = v.y, x[e + 2] = v.z, x[e + 3] = v.w;
            }
        } else {
            static_assert(E == 8, "16 bytes of half types");
            const uint4 v = *(const uint4 *)((const unsigned short *)row + i);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++) x[2 * e] = widen_act(w[e] & 0xffff, SRC), x[2 * e + 1] = widen_act(w[e] >> 16, SRC);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = i + e >= from && i + e < end ? load_act(row, i + e, SRC) : none;
}
// A row of f32 that is not aligned as the other one is
template <int E> __device__ __forceinline__ void load_apart(float *x, const float *row, uint32_t i, uint32_t from, uint32_t end) {
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = i + e >= from && i + e < end ? row[i + e - from] : 0.0f;
}

// CTAS_SM: 1, or where there are more CTAs than SMs 2, so that one request's weights are formed while another one's CTAs wait for each other (64 trees over 128256 tokens 106.9 and 93.9 us, one chain 24.3 and 25.6)
template <int SRC, int CTAS_SM> __global__ void __launch_bounds__(THREADS, CTAS_SM) paged_verify_kernel(const PagedVerifyArgs a, uint32_t ctas, uint32_t part) {
    constexpr uint32_t BATCH = 16 / CTAS_SM, FAST = 32 / CTAS_SM;  // tokens that a thread has in flight in a pass of 64 and of 32 bits
    constexpr int E = SRC == ACT_F32 ? 4 : 8, U = BATCH / E, V = FAST / E;
    constexpr uint32_t EB = act_elem_bytes(SRC);
    extern __shared__ __align__(16) uint8_t smem[];
    Shared &sh = *(Shared *)smem;
    const uint32_t most = a.s.max_new;
    Node *const node = (Node *)(smem + sizeof(Shared));
    double *const value = (double *)(node + most);                        // what is left of a child's weight
    double *const taken = value + most;                                   // sums in front of the rejections: each takes the draft's share of its one from every weight
    int32_t *const parent = (int32_t *)(taken + most);
    uint32_t *const gone = (uint32_t *)(parent + most);                   // bits of the CTA's places
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cluster_rank();
    const uint32_t me = rank * WARPS + warp, warps = ctas * WARPS;        // of the cluster's warps
    const uint32_t first = me * part, part0 = rank * WARPS * part;        // the warp's places, the CTA's
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (tid < 16) sh.root[tid] = exp2((double)tid / 16.0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t set = 0;
    const bool fits = *a.stamped == a.stamp;
    if (!fits && blockIdx.x == 0 && tid == 0 && a.status) atomicOr(a.status, (int)PAGED_STATUS_PLAN);

    auto warp_sum = [&](auto s) {
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    };
    // Where running sums over the lanes' parts, `front` in front of them, pass `goal`: the part (32: none has a weight) and the sum in front of it. Where none does, by a rounding, it is the
    // last part with a weight.
    auto place_of = [&](double own, double front, double goal, double &before) -> uint32_t {
        double inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const uint32_t some = __ballot_sync(0xffffffffu, own > 0.0), past = __ballot_sync(0xffffffffu, own > 0.0 && front + inc > goal);
        if (!some) return 32;
        const uint32_t at = past ? __ffs(past) - 1 : 31 - __clz(some);
        before = __shfl_sync(0xffffffffu, front + (inc - own), at);
        return at;
    };

    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all of them are there: their memory may be written
    __syncthreads();
    const uint32_t clusters = gridDim.x / ctas;
#pragma unroll 1
    for (uint32_t r = blockIdx.x / ctas; r < a.s.requests; r += clusters) {
        const uint4 rec = ((const uint4 *)a.request)[r];
        // (what decides is rank 0's; where the others' own differ, since the caller writes them meanwhile, only numbers do)
        const float own_temperature = a.temperature ? a.temperature[r] : 1.0f;
        const uint32_t q0 = rec.x, own_n = fits ? min(rec.y - rec.x, most) : 0;
        uint32_t n = own_n;
        bool cold = !(own_temperature > 0.0f);
        float temperature = own_temperature;
        uint32_t v = 0, length = 0;
        int32_t answer = -1;
        for (;;) {  // a level
            const char *const start = (const char *)a.logits + (q0 + v) * a.logits_row * EB;
            const uint32_t from = (uint32_t)((uintptr_t)start & 15) / EB, end = from + a.vocab, last = own_n ? min(first + part, end) : 0u;
            const char *const row = start - from * EB;
            const float *const draft = a.draft ? a.draft + (q0 + v) * a.draft_row : nullptr;
            const bool same = ((uintptr_t)(draft - from) & 15) == 0;
            // ---- the largest logit, and the sum of the weights in 32 bits, relative to each thread's largest
            float x[V][E];
            auto fetch = [&](uint32_t c0) {
#pragma unroll
                for (int u = 0; u < V; u++) {
                    const uint32_t i = c0 + lane * E + 32 * E * u;
                    if (i < last) load_row<SRC, E>(x[u], row, i, from, end, -INFINITY);
                    else
#pragma unroll
                        for (int e = 0; e < E; e++) x[u][e] = -INFINITY;
                }
            };
            fetch(first);
            // (meanwhile rank 0 fetches what the tests of the children need, a thread for a token)
            if (rank == 0 && length == 0) {
#pragma unroll 1
                for (uint32_t t = tid; t < n; t += THREADS) {
                    const int32_t p = a.parents ? a.parents[q0 + t] : (int32_t)t - 1, token = a.tokens[q0 + t];
                    const float accept = a.accept[q0 + t];
                    parent[t] = p, node[t].token = token, node[t].accept = accept;
#pragma unroll 1
                    for (uint32_t c = 1; c < ctas; c++) {
                        put(of_rank(parent + t, c), (uint32_t)p);
                        put(of_rank(node + t, c), (uint64_t)(uint32_t)token | (uint64_t)__float_as_uint(accept) << 32);
                    }
                }
                if (tid < ctas) put(of_rank(&sh.n, tid), n), put(of_rank(&sh.temperature, tid), own_temperature);
            }
            float child_logit = 0.0f, child_draft = 0.0f;
            auto is_child = [&](uint32_t t) { return t > v && t < n && parent[t] == (int32_t)v; };
            auto fetch_child = [&](uint32_t t) {
                if (!is_child(t)) return;
                const uint32_t token = (uint32_t)node[t].token;
                if (token >= a.vocab) {
                    if (a.status) atomicOr(a.status, (int)PAGED_STATUS_INDEX);
                    return;
                }
                child_logit = load_act(start, token, SRC);
                if (draft) child_draft = draft[token];
            };
            auto tell_child = [&](uint32_t t) {  // (a lane for a CTA)
                uint32_t children = __ballot_sync(0xffffffffu, is_child(t));
                while (children) {
                    const uint32_t who = __ffs(children) - 1;
                    children &= children - 1;
                    const float x = __shfl_sync(0xffffffffu, child_logit, who), y = __shfl_sync(0xffffffffu, child_draft, who);
                    if (lane < ctas) put(of_rank(&node[t - lane + who].logit, lane), (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32);
                }
            };
            if (rank == 0) {
#pragma unroll 1
                for (uint32_t t0 = THREADS; t0 < n; t0 += THREADS) fetch_child(t0 + tid), tell_child(t0 + tid);
                fetch_child(tid);
            }
            const float scale = fminf(fmaxf(1.44269504f / temperature, 1e-45f), 3e38f);  // (not 0, not infinite: -inf times it is -inf, 0 times it 0)
            float top = -INFINITY, sum = 0.0f;
            uint32_t at = ~0u;
#pragma unroll 1
            for (uint32_t c0 = first; c0 < last;) {
                if (cold) {
#pragma unroll
                    for (int u = 0; u < V; u++)
                        if (c0 + 32 * E * u < last)
#pragma unroll
                            for (int e = 0; e < E; e++) better(top, at, x[u][e], c0 + lane * E + 32 * E * u + e);
                } else {
                    float largest[4] = {top, top, top, top};
#pragma unroll
                    for (int u = 0; u < V; u++)
                        if (c0 + 32 * E * u < last)
#pragma unroll
                            for (int e = 0; e < E; e++) largest[e & 3] = max_nan(largest[e & 3], x[u][e]);
                    const float was = top;
                    top = max_nan(max_nan(largest[0], largest[1]), max_nan(largest[2], largest[3]));
                    if (top != -INFINITY) {
                        sum *= exp2_fast((was - top) * scale);
                        float s[4] = {};
#pragma unroll
                        for (int u = 0; u < V; u++)
                            if (c0 + 32 * E * u < last)
#pragma unroll
                                for (int e = 0; e < E; e++) s[e & 3] += exp2_fast((x[u][e] - top) * scale);
                        sum += (s[0] + s[1]) + (s[2] + s[3]);
                    }
                }
                c0 += 32 * FAST;
                if (c0 < last) fetch(c0);
            }
            {
                const float mine = top;
                uint64_t told;
                top = unordered(__reduce_max_sync(0xffffffffu, ordered(top)));
                if (cold) {
                    at = __reduce_min_sync(0xffffffffu, mine == top ? at : ~0u);
                    told = (uint64_t)ordered(top) << 32 | (uint32_t)~at;
                } else {
                    sum = warp_sum(mine == -INFINITY ? 0.0f : sum * exp2_fast((mine - top) * scale));
                    told = (uint64_t)__float_as_uint(sum) << 32 | __float_as_uint(top);
                }
                if (lane < ctas) put(of_rank(&sh.quick[set][me], lane), told);
            }
            if (rank == 0) tell_child(tid);
            cluster_sync();
            if (length == 0) {
                n = sh.n;
                temperature = sh.temperature;
                cold = !(temperature > 0.0f);
                if (n == 0) break;
                if (rank == 0 && tid == 0) a.path[(size_t)r * most] = 0;
                length = 1;
            }
            uint32_t best = 0;  // the token of the largest logit
            if (cold) {
                uint32_t hi = 0, lo = 0;
#pragma unroll
                for (uint32_t k = 0; k < MOST_CTAS * WARPS / 32; k++) {
                    const uint64_t q = lane + 32 * k < warps ? sh.quick[set][lane + 32 * k] : 0;
                    if ((uint32_t)(q >> 32) > hi || ((uint32_t)(q >> 32) == hi && (uint32_t)q > lo)) hi = (uint32_t)(q >> 32), lo = (uint32_t)q;
                }
                const uint32_t most_hi = __reduce_max_sync(0xffffffffu, hi);
                best = ~__reduce_max_sync(0xffffffffu, hi == most_hi ? lo : 0u) - from;
                top = unordered(most_hi);
            } else {
                float mine = -INFINITY, tops[MOST_CTAS * WARPS / 32], parts_of[MOST_CTAS * WARPS / 32];
#pragma unroll
                for (uint32_t k = 0; k < MOST_CTAS * WARPS / 32; k++) {
                    const uint64_t q = lane + 32 * k < warps ? sh.quick[set][lane + 32 * k] : 0x00000000ff800000ull;
                    tops[k] = __uint_as_float((uint32_t)q), parts_of[k] = __uint_as_float((uint32_t)(q >> 32));
                    mine = max_nan(mine, tops[k]);
                }
                top = unordered(__reduce_max_sync(0xffffffffu, ordered(mine)));
                sum = 0.0f;
#pragma unroll
                for (uint32_t k = 0; k < MOST_CTAS * WARPS / 32; k++) sum = fmaf(parts_of[k], exp2_fast((tops[k] - top) * scale), sum);
                sum = warp_sum(sum);
            }
            set ^= 1;
            if (!(top < INFINITY) || top == -INFINITY) {  // NaN, +inf, or nothing at all
                if (rank == 0 && tid == 0 && a.status) atomicOr(a.status, (int)PAGED_STATUS_LOGITS);
                break;
            }
            // ---- the children
            uint32_t next = 0, stages = 0;       // the accepted child (0: none), rejections that took something
            bool exact = false, parts = false;   // in 64 bits from here on; the last exchange's sums are those of what is left
            double rest = (double)sum;           // what the distribution's weights add up to,
            double full = rest, unsure = SURE;   // and did before tokens left it; how far off that may be
            Weight weight(sh.root, top);
            uint32_t t = v + 1;
            for (;;) {
                while (t < n && (parent[t] != (int32_t)v || (uint32_t)node[t].token >= a.vocab)) t++;
                if (cold) {
                    if (t == n) break;
                    if ((uint32_t)node[t].token == best) {
                        next = t;
                        break;
                    }
                    t++;
                    continue;
                }
                if (!exact) {
                    if (t < n) {  // most children's tests need no more than 32 bits
                        const Node y = node[t];
                        const float line = (draft ? y.accept * y.draft : y.accept) * sum, mine = exp2_fast((y.logit - top) * scale);
                        if (mine - line > fmaxf(mine * (float)SURE, 1e-30f)) {
                            next = t;
                            break;
                        }
                    }
                    exact = true;
                    weight.set(temperature);
#pragma unroll 1
                    for (uint32_t k = v + 1 + tid; k < n; k += THREADS)
                        if (parent[k] == (int32_t)v) value[k] = weight(node[k].logit);
                    if (!draft)
#pragma unroll 1
                        for (uint32_t i = tid; i < WARPS * part / 32; i += THREADS) gone[i] = 0;
                    __syncthreads();
                }
                // the child's test; what is to be added up next: nothing (the next child), what is left, or what the draft leaves of that
                bool minus = false, again = false;
                if (t < n) {
                    const Node y = node[t];
                    const double u = draft ? (double)y.accept * (double)y.draft : (double)y.accept, line = u * rest, mine = value[t];
                    again = unsure != 0.0 && !(fabs(line - mine) > fabs(u) * full * SURE);
                    if (!again) {
                        if (line < mine) {
                            next = t;
                            break;
                        }
                        if (draft) {
                            again = unsure != 0.0;  // (what it leaves depends on the sum)
                            minus = !again;
                        } else {
                            t++;
                            if (!(mine > 0.0)) continue;
                            __syncthreads();  // (value[] has been read)
#pragma unroll 1
                            for (uint32_t k = t - 1 + tid; k < n; k += THREADS)
                                if (parent[k] == (int32_t)v && node[k].token == y.token) value[k] = 0.0;
                            const uint32_t bit = (uint32_t)y.token + from - part0;
                            if (tid == 0 && bit < WARPS * part) gone[bit >> 5] |= 1u << (bit & 31);
                            __syncthreads();
                            rest -= weight(y.logit);
                            if (rest > full * 0x1p-10) continue;
                            again = true;  // what is left was lost in the difference
                        }
                    }
                } else if (parts) {
                    break;
                }
                double s2[2] = {};
#pragma unroll 1
                for (uint32_t i0 = first + lane * E; i0 < last; i0 += 32 * BATCH) {
                    float z[U][E], d[U][E];
                    double w[BATCH];
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const uint32_t i = i0 + 32 * E * u;
#pragma unroll
                        for (int e = 0; e < E; e++) z[u][e] = -INFINITY, d[u][e] = 0.0f;
                        if (i >= last) continue;
                        load_row<SRC, E>(z[u], row, i, from, end, -INFINITY);
                        if (draft && (stages || minus)) {
                            if (same) load_row<ACT_F32, E>(d[u], draft - from, i, from, end, 0.0f);
                            else load_apart<E>(d[u], draft, i, from, end);
                        }
                    }
                    if (!draft)
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const uint32_t i = i0 + 32 * E * u, bits = i < last ? gone[(i - part0) >> 5] >> (i & 31) : 0u;
                            if (bits & ((1u << E) - 1))
#pragma unroll
                                for (int e = 0; e < E; e++) z[u][e] = bits >> e & 1 ? -INFINITY : z[u][e];
                        }
#pragma unroll
                    for (int e = 0; e < (int)BATCH; e++) w[e] = weight(z[e / E][e % E]);
#pragma unroll 1
                    for (uint32_t k = 0; k < stages; k++) {
                        const double share = -taken[k];
#pragma unroll
                        for (int e = 0; e < (int)BATCH; e++) w[e] = positive(fma((double)d[e / E][e % E], share, w[e]));
                    }
                    if (minus) {
#pragma unroll
                        for (int e = 0; e < (int)BATCH; e++) w[e] = positive(fma((double)d[e / E][e % E], -rest, w[e]));
                    }
#pragma unroll
                    for (int e = 0; e < (int)BATCH; e++) s2[e & 1] += w[e];
                }
                const double own = warp_sum(s2[0] + s2[1]);
                if (lane < ctas) put(of_rank(&sh.sum[set][me], lane), own);
                cluster_sync();
                double left2[2] = {};
#pragma unroll
                for (uint32_t k = 0; k < MOST_CTAS * WARPS / 32; k++) left2[k & 1] += lane + 32 * k < warps ? sh.sum[set][lane + 32 * k] : 0.0;
                const double left = warp_sum(left2[0] + left2[1]);
                set ^= 1;
                if (minus) {
                    t++;
                    parts = left > 0.0;
                    if (!parts) continue;  // (nothing is left, and the distribution stays)
#pragma unroll 1
                    for (uint32_t k = t + tid; k < n; k += THREADS)
                        if (parent[k] == (int32_t)v) value[k] = positive(fma((double)node[k].draft, -rest, value[k]));
                    if (tid == 0) taken[stages] = rest;
                    stages++;
                    rest = left;
                    __syncthreads();
                    continue;
                }
                rest = full = left;
                unsure = 0.0;
                if (!again) break;
            }
            if (next) {
                if (rank == 0 && tid == 0) a.path[(size_t)r * most + length] = (int32_t)next;
                v = next;
                length++;
                continue;
            }
            // ---- no child: the token behind the path
            if (cold) {
                answer = (int32_t)best;
                break;
            }
            // the warp whose tokens the number falls among, from the warps' sums (a lane has some behind each other); its lanes' tokens, then
            const double goal = (double)a.pick[r] * rest;
            const double *const sums = sh.sum[set ^ 1];
            const uint32_t each = (warps + 31) / 32;
            double before = 0.0, mine = 0.0;
#pragma unroll 1
            for (uint32_t k = 0; k < each; k++) mine += lane * each + k < warps ? sums[lane * each + k] : 0.0;
            uint32_t who = place_of(mine, 0.0, goal, before);
            answer = who < 32 ? -2 : -1;  // (-2: written by that warp)
            if (who < 32) {
                const uint32_t begin = who * each;
                double run = before;
                who = begin;
#pragma unroll 1
                for (uint32_t k = begin; k < min(begin + each, warps); k++) {
                    if (sums[k] > 0.0) who = k, before = run;
                    run += sums[k];
                    if (sums[k] > 0.0 && run > goal) break;
                }
                if (who == me) {
                    uint32_t token = 0;
                    bool found = false;
#pragma unroll 1
                    for (uint32_t c0 = first; c0 < last && !found; c0 += 32 * BATCH) {  // a lane has BATCH tokens behind each other
                        const uint32_t i0 = c0 + lane * BATCH;
                        float z[U][E], d[U][E];
                        double wt[BATCH], own = 0.0;
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const uint32_t i = i0 + E * u;
#pragma unroll
                            for (int e = 0; e < E; e++) z[u][e] = -INFINITY, d[u][e] = 0.0f;
                            if (i >= last) continue;
                            load_row<SRC, E>(z[u], row, i, from, end, -INFINITY);
                            if (!draft) {
                                const uint32_t bits = gone[(i - part0) >> 5] >> (i & 31);
#pragma unroll
                                for (int e = 0; e < E; e++) z[u][e] = bits >> e & 1 ? -INFINITY : z[u][e];
                            } else if (stages) {
                                if (same) load_row<ACT_F32, E>(d[u], draft - from, i, from, end, 0.0f);
                                else load_apart<E>(d[u], draft, i, from, end);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < (int)BATCH; e++) wt[e] = weight(z[e / E][e % E]);
#pragma unroll 1
                        for (uint32_t k = 0; k < stages; k++) {
                            const double share = -taken[k];
#pragma unroll
                            for (int e = 0; e < (int)BATCH; e++) wt[e] = positive(fma((double)d[e / E][e % E], share, wt[e]));
                        }
#pragma unroll
                        for (int e = 0; e < (int)BATCH; e++) own += wt[e];
                        const uint32_t l = place_of(own, before, goal, before);
                        if (l == 32) continue;
                        // (the lane's first token past the goal, else its last one with a weight)
                        double past_sum = before;
                        uint32_t at_last = 0;
                        bool past = false;
#pragma unroll
                        for (int e = 0; e < (int)BATCH; e++) {
                            past_sum += wt[e];
                            if (wt[e] > 0.0 && !past) at_last = i0 + e, past = past_sum > goal;
                        }
                        token = __shfl_sync(0xffffffffu, at_last, l);
                        before = __shfl_sync(0xffffffffu, past_sum, l);
                        found = __shfl_sync(0xffffffffu, (int)past, l);
                    }
                    if (lane == 0) a.next[r] = (int32_t)(token - from);
                }
            }
            break;
        }
        if (rank == 0) {
            if (tid == 0) {
                a.accepted[r] = (int32_t)length;
                if (answer != -2) a.next[r] = answer;
            }
#pragma unroll 1
            for (uint32_t i = length + tid; i < most; i += THREADS) a.path[(size_t)r * most + i] = -1;
        }
        cluster_sync();  // the request's nodes have been read by all
    }
}

}  // namespace pv

// A warp's places with so many CTAs a request, whole vectors of all its lanes
static uint32_t verify_part(const PagedVerifyArgs &a, uint32_t ctas) {
    const uint32_t E = 16 / act_elem_bytes(a.type), unit = 32 * E, warps = ctas * pv::WARPS, places = a.vocab + E - 1;  // (a row may begin inside a vector)
    return ((places + warps - 1) / warps + unit - 1) / unit * unit;
}

template <int SRC, int CTAS_SM> static cudaError_t verify_launch(const PagedVerifyArgs &a, uint32_t ctas, int sm_count, bool pdl, cudaStream_t stream) {
    auto *kernel = pv::paged_verify_kernel<SRC, CTAS_SM>;
    static std::once_flag once[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::call_once(once[dev & 63], [&] {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pv::SMEM_MOST);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (e != cudaSuccess) return e;
    const uint32_t part = verify_part(a, ctas);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    const uint32_t clusters = std::min<uint32_t>(a.s.requests, std::max<uint32_t>(1, CTAS_SM * (uint32_t)sm_count / ctas));
    cfg.gridDim = dim3(clusters * ctas);
    cfg.blockDim = dim3(pv::THREADS);
    cfg.dynamicSmemBytes = pv::shared_bytes(a.s.max_new, part);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, ctas, part);
}

cudaError_t launch_paged_verify(const PagedVerifyArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    // As many CTAs a request as leave a warp 500 tokens, and no more than two for each SM in all, of 16 one: one chain over 128256 tokens with 4, 8, 16 CTAs 41.0, 28.5, 24.3 us; 16 trees over 32000 with 2, 4, 8 26.0,
    // 21.3, 27.8; over 128256 16 trees with 8 and 16 44.0 and 50.7, 24 and 32 trees with 4, 8, 16 66, 61, 68 and 67, 63, 83, 64 trees with 2, 4, 8 114, 97, 107
    uint32_t ctas = pv::MOST_CTAS;
    while (ctas > 1 && ((uint64_t)a.s.requests * ctas > (ctas > 8 ? 1 : 2) * (uint64_t)sm_count || a.vocab < 500 * pv::WARPS * ctas)) ctas /= 2;
    while (ctas < pv::MOST_CTAS && verify_part(a, ctas) > pv::PART_MOST) ctas *= 2;
    const bool many = (uint64_t)a.s.requests * ctas > (uint64_t)sm_count;
    auto run = [&](auto src) {
        constexpr int S = decltype(src)::value;
        return many ? verify_launch<S, 2>(a, ctas, sm_count, pdl, stream) : verify_launch<S, 1>(a, ctas, sm_count, pdl, stream);
    };
    return a.type == ACT_F32 ? run(std::integral_constant<int, ACT_F32>()) : a.type == ACT_F16 ? run(std::integral_constant<int, ACT_F16>()) : run(std::integral_constant<int, ACT_BF16>());
}

}  // namespace lb
