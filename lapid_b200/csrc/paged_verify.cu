// Which drafted tokens the model's probabilities accept, and the token behind them.
//
// A request's first token is the text's last; its logits z give the distribution of what follows, P = softmax(z / T) (T = 0: the largest alone). The walk begins there. The
// children of the node v it has reached are tried in their order: with the draft's distribution D of v, child c with token x is accepted when u_c D(x) < P(x), else P becomes what D
// left, max(P - D, 0) / sum of it; without D (candidates that were chosen, not drawn) when u_c < P(x), else x leaves P. An accepted child is the next v; when none is,
// the token behind the path is the first t with P(0) + .. + P(t) > w. Whatever the drafts are, the tokens are then distributed as the model's own.
//
// Decisions are comparisons, so weights and sums are 64 bits wide: a result differs from the definition's only where u or w is within 1e-13 of a border.
//
// A request belongs to a cluster of CTAs, each with a part of the vocabulary, a warp of it 32 vectors wide and so on to its end; only the rows on the path are read. A level is a pass over the
// node's logits (largest and sum, each thread relative to its own largest), an exchange over the cluster's shared memory, and the children's tests, whose tokens, numbers and values were
// fetched meanwhile. What decides comes from rank 0's loads and from the exchanged sums alone, so that the CTAs of a cluster always take the same way.
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

constexpr uint32_t WARPS = 16, THREADS = 32 * WARPS, MOST_CTAS = 8;  // of a cluster
constexpr int UNROLL = 4;                                             // vectors a thread has in flight

// Shared memory: what the exchanges bring (two sets: a CTA writes a set again only when all have read it, which they say with the exchange between), the request, its
// nodes, and a bit for each token of the part that is out of the distribution.
struct Exchange {
    double sum[2][MOST_CTAS];
    float top[2][MOST_CTAS];
    uint32_t at[2][MOST_CTAS];
};
struct Shared {
    Exchange ex;
    double warp_sum[WARPS];
    float warp_top[WARPS];
    uint32_t warp_at[WARPS];
    uint32_t n;
    float temperature;
};
struct Node {      // what rank 0 tells of a child
    int32_t token;
    float accept, logit, draft;
};

// value, inverse, node and parent of each of `most` tokens, and a bit for each token of the vocabulary's part
constexpr size_t shared_bytes(uint32_t most, uint32_t part) { return sizeof(Shared) + most * (2 * sizeof(double) + sizeof(Node) + 4) + (size_t)WARPS * part / 8; }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t of_rank(const void *p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(s32(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void put(uint32_t at, uint32_t x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); }
__device__ __forceinline__ void put(uint32_t at, float x) { put(at, __float_as_uint(x)); }
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

// e^((z - top) / T): 0 for -inf, whatever T is
__device__ __forceinline__ double weight(float z, float top, double inv_t) { return z == -INFINITY ? 0.0 : exp(((double)z - (double)top) * inv_t); }

// E elements of a row from `i` (a multiple of E) on; `none` behind the vocabulary
template <int SRC, int E, bool VEC> __device__ __forceinline__ void load_row(float (&x)[E], const void *row, uint32_t i, uint32_t vocab, float none) {
    if (VEC && i + E <= vocab) {
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
    for (int e = 0; e < E; e++) x[e] = i + e < vocab ? load_act(row, i + e, SRC) : none;
}

template <int SRC, bool VEC> __global__ void __launch_bounds__(THREADS, 2) paged_verify_kernel(const PagedVerifyArgs a, uint32_t ctas, uint32_t part) {
    constexpr int E = SRC == ACT_F32 ? 4 : 8;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared &sh = *(Shared *)smem;
    const uint32_t most = a.s.max_new;
    double *const value = (double *)(smem + sizeof(Shared));              // a child's P(x), kept up with what is taken from P
    double *const inverse = value + most;                                 // 1 / sum of what the draft left, a rejection each
    Node *const node = (Node *)(inverse + most);
    int32_t *const parent = (int32_t *)(node + most);
    uint32_t *const gone = (uint32_t *)(parent + most);                   // bits of the part's tokens
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cluster_rank();
    const uint32_t first = (rank * WARPS + warp) * part, last = min(first + part, a.vocab);  // the warp's tokens
    const uint32_t part0 = rank * WARPS * part, part_words = WARPS * part / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint32_t set = 0;
    const bool fits = *a.stamped == a.stamp;
    if (!fits && blockIdx.x == 0 && tid == 0 && a.status) atomicOr(a.status, (int)PAGED_STATUS_PLAN);

    // ---- what the CTAs exchange
    auto warp_sum = [&](double s) {
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    };
    // The sum over the cluster of the threads' sums, in the ranks' order; warp_sum[] keeps the warps'
    auto exchange_sum = [&](double s, double *before_rank = nullptr) -> double {
        s = warp_sum(s);
        if (lane == 0) sh.warp_sum[warp] = s;
        __syncthreads();
        if (warp == 0 && lane < ctas) {
            double t = 0.0;
            for (uint32_t w = 0; w < WARPS; w++) t += sh.warp_sum[w];
            put(of_rank(&sh.ex.sum[set][rank], lane), t);
        }
        cluster_sync();
        double all = 0.0;
        for (uint32_t c = 0; c < ctas; c++) {
            if (before_rank) before_rank[c] = all;
            all += sh.ex.sum[set][c];
        }
        set ^= 1;
        return all;
    };

    cluster_sync();  // (all of them are there: their memory may be written)
    const uint32_t clusters = gridDim.x / ctas;
    for (uint32_t r = blockIdx.x / ctas; r < a.s.requests; r += clusters) {
        const uint4 rec = ((const uint4 *)a.request)[r];
        const uint32_t q0 = rec.x;
        if (rank == 0) {
            const uint32_t n = fits ? min(rec.y - rec.x, most) : 0;
            const float temperature = a.temperature ? a.temperature[r] : 1.0f;
            for (uint32_t t = tid; t < n; t += THREADS) {
                const int32_t p = a.parents ? a.parents[q0 + t] : (int32_t)t - 1;
                for (uint32_t c = 0; c < ctas; c++) put(of_rank(parent + t, c), (uint32_t)p);
            }
            if (tid < ctas) put(of_rank(&sh.n, tid), n), put(of_rank(&sh.temperature, tid), temperature);
        }
        cluster_sync();
        const uint32_t n = sh.n;
        const float temperature = sh.temperature;
        const bool cold = !(temperature > 0.0f);
        const double inv_t = cold ? 0.0 : 1.0 / (double)temperature;
        uint32_t v = 0, length = n ? 1 : 0;
        int32_t answer = -1;
        if (n && rank == 0 && tid == 0) a.path[(size_t)r * most] = 0;
        while (n) {
            // ---- rank 0 fetches what the children's tests need
            const char *const row = (const char *)a.logits + (q0 + v) * a.logits_row * act_elem_bytes(SRC);
            const float *const draft = a.draft ? a.draft + (q0 + v) * a.draft_row : nullptr;
            if (rank == 0) {
                for (uint32_t t = v + 1 + tid; t < n; t += THREADS) {
                    if (parent[t] != (int32_t)v) continue;
                    Node x{a.tokens[q0 + t], a.accept[q0 + t], 0.0f, 0.0f};
                    if ((uint32_t)x.token < a.vocab) {
                        x.logit = load_act(row, (uint32_t)x.token, SRC);
                        if (draft) x.draft = draft[x.token];
                    } else {
                        if (a.status) atomicOr(a.status, (int)PAGED_STATUS_INDEX);
                        x.token = -1;  // (never accepted)
                    }
                    for (uint32_t c = 0; c < ctas; c++) {
                        const uint32_t to = of_rank(node + t, c);
                        put(to, (uint32_t)x.token), put(to + 4, x.accept), put(to + 8, x.logit), put(to + 12, x.draft);
                    }
                }
            }
            // ---- the largest logit and the sum of the weights
            float top = -INFINITY;
            uint32_t at = ~0u;
            double sum = 0.0;
            for (uint32_t i0 = first + lane * E; i0 < last; i0 += 32 * E * UNROLL) {
                float x[UNROLL][E];
#pragma unroll
                for (int u = 0; u < UNROLL; u++) {
                    const uint32_t i = i0 + 32 * E * u;
                    if (i < last) load_row<SRC, E, VEC>(x[u], row, i, a.vocab, -INFINITY);
                    else
#pragma unroll
                        for (int e = 0; e < E; e++) x[u][e] = -INFINITY;
                }
                const float was = top;
#pragma unroll
                for (int u = 0; u < UNROLL; u++)
#pragma unroll
                    for (int e = 0; e < E; e++) better(top, at, x[u][e], i0 + 32 * E * u + e);
                if (cold || top == -INFINITY) continue;
                if (top != was) sum *= weight(was, top, inv_t);
#pragma unroll
                for (int u = 0; u < UNROLL; u++)
#pragma unroll
                    for (int e = 0; e < E; e++) sum += weight(x[u][e], top, inv_t);
            }
            const float mine = top;
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const float t = __shfl_xor_sync(0xffffffffu, top, o);
                better(top, at, t, __shfl_xor_sync(0xffffffffu, at, o));
            }
            sum = warp_sum(sum * weight(mine, top, inv_t));
            if (lane == 0) sh.warp_top[warp] = top, sh.warp_at[warp] = at, sh.warp_sum[warp] = sum;
            __syncthreads();
            if (warp == 0 && lane < ctas) {
                top = -INFINITY, at = ~0u;
                for (uint32_t w = 0; w < WARPS; w++) better(top, at, sh.warp_top[w], sh.warp_at[w]);
                sum = 0.0;
                for (uint32_t w = 0; w < WARPS; w++) sum += sh.warp_sum[w] * weight(sh.warp_top[w], top, inv_t);
                put(of_rank(&sh.ex.sum[set][rank], lane), sum);
                put(of_rank(&sh.ex.top[set][rank], lane), top);
                put(of_rank(&sh.ex.at[set][rank], lane), at);
            }
            cluster_sync();
            top = -INFINITY, at = ~0u;
            for (uint32_t c = 0; c < ctas; c++) better(top, at, sh.ex.top[set][c], sh.ex.at[set][c]);
            double total = 0.0;
            for (uint32_t c = 0; c < ctas; c++) total += sh.ex.sum[set][c] * weight(sh.ex.top[set][c], top, inv_t);
            set ^= 1;
            if (!(top < INFINITY) || top == -INFINITY) {  // NaN, +inf, or nothing at all
                if (rank == 0 && tid == 0 && a.status) atomicOr(a.status, (int)PAGED_STATUS_LOGITS);
                break;
            }
            // ---- the children
            const double inv_total = 1.0 / total;
            for (uint32_t t = v + 1 + tid; t < n; t += THREADS)
                if (parent[t] == (int32_t)v) {
                    const Node x = node[t];
                    value[t] = x.token < 0 ? 0.0 : cold ? ((uint32_t)x.token == at ? 1.0 : 0.0) : weight(x.logit, top, inv_t) * (draft ? inv_total : 1.0);
                }
            if (!draft && !cold)
                for (uint32_t i = tid; i < part_words; i += THREADS) gone[i] = 0;
            __syncthreads();
            uint32_t next = 0, stages = 0;  // the accepted child (0: none), rejections that took something
            double rest = total;            // without a draft: what the distribution's weights add up to
            // what is left of a token with weight w and draft probability d
            auto left = [&](double w, double d) {
                w *= inv_total;
                for (uint32_t k = 0; k < stages; k++) w = fmax(w - d, 0.0) * inverse[k];
                return w;
            };
            // f(token, weight left) over the warp's tokens, in their order within a thread
            auto over = [&](auto &&f) {
                for (uint32_t i = first + lane * E; i < last; i += 32 * E) {
                    float x[E], d[E];
                    load_row<SRC, E, VEC>(x, row, i, a.vocab, -INFINITY);
                    if (draft) load_row<ACT_F32, E, VEC>(d, draft, i, a.vocab, 0.0f);
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        double w = weight(x[e], top, inv_t);
                        if (draft) w = left(w, (double)d[e]);
                        else if (gone[(i + e - part0) >> 5] >> ((i + e) & 31) & 1) w = 0.0;
                        f(w, draft ? (double)d[e] : 0.0);
                    }
                }
            };
            for (uint32_t t = v + 1; t < n && !next; t++) {
                if (parent[t] != (int32_t)v) continue;
                const Node x = node[t];
                if (x.token < 0) continue;
                if (cold) {
                    if ((uint32_t)x.token == at) next = t;
                } else if (draft) {
                    if ((double)x.accept * (double)x.draft < value[t]) {
                        next = t;
                    } else {
                        double s = 0.0;
                        over([&](double w, double d) { s += fmax(w - d, 0.0); });
                        s = exchange_sum(s);
                        if (s > 0.0) {  // (else nothing is left, and the distribution stays)
                            const double inv = 1.0 / s;
                            for (uint32_t j = t + 1 + tid; j < n; j += THREADS)
                                if (parent[j] == (int32_t)v) value[j] = fmax(value[j] - (double)node[j].draft, 0.0) * inv;
                            if (tid == 0) inverse[stages] = inv;
                            stages++;
                            __syncthreads();
                        }
                    }
                } else {
                    if ((double)x.accept * rest < value[t]) {
                        next = t;
                    } else if (value[t] > 0.0) {
                        __syncthreads();  // (value[] has been read)
                        for (uint32_t j = t + tid; j < n; j += THREADS)
                            if (parent[j] == (int32_t)v && node[j].token == x.token) value[j] = 0.0;
                        const uint32_t bit = (uint32_t)x.token - part0;
                        if (tid == 0 && (uint32_t)x.token >= part0 && bit < WARPS * part) gone[bit >> 5] |= 1u << (bit & 31);
                        __syncthreads();
                        rest -= weight(x.logit, top, inv_t);
                        if (!(rest > total * 0x1p-10)) {  // what is left was lost in the difference: add it up
                            double s = 0.0;
                            over([&](double w, double) { s += w; });
                            rest = exchange_sum(s);
                        }
                    }
                }
            }
            if (next) {
                if (rank == 0 && tid == 0) a.path[(size_t)r * most + length] = (int32_t)next;
                v = next;
                length++;
                continue;
            }
            // ---- no child: the token behind the path
            if (cold) {
                answer = (int32_t)at;
                break;
            }
            double s = 0.0, before[MOST_CTAS];
            over([&](double w, double) { s += w; });
            const double all = exchange_sum(s, before);
            const double goal = (double)a.pick[r] * all;
            uint32_t who = ctas;
            for (uint32_t c = 0; c < ctas; c++) {
                const double own = sh.ex.sum[set ^ 1][c];
                if (own > 0.0 && (who == ctas || !(before[who] + sh.ex.sum[set ^ 1][who] > goal))) who = c;
            }
            if (who == rank) {
                double front = before[rank];
                uint32_t w = WARPS;
                double w_front = front;
                for (uint32_t i = 0; i < WARPS; i++) {
                    const double own = sh.warp_sum[i];
                    if (own > 0.0 && (w == WARPS || !(w_front + sh.warp_sum[w] > goal))) w = i, w_front = front;
                    front += own;
                }
                if (w == warp) {
                    double run = w_front;
                    uint32_t found = ~0u, some = ~0u;  // the first past the goal, the last with a weight
                    for (uint32_t i0 = first; i0 < last && found == ~0u; i0 += 32 * E) {
                        const uint32_t i = i0 + lane * E;
                        float x[E], d[E];
                        double wt[E], mine = 0.0;
#pragma unroll
                        for (int e = 0; e < E; e++) x[e] = -INFINITY, d[e] = 0.0f;
                        if (i < last) {
                            load_row<SRC, E, VEC>(x, row, i, a.vocab, -INFINITY);
                            if (draft) load_row<ACT_F32, E, VEC>(d, draft, i, a.vocab, 0.0f);
                        }
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            wt[e] = weight(x[e], top, inv_t);
                            if (draft) wt[e] = left(wt[e], (double)d[e]);
                            else if (i < last && gone[(i + e - part0) >> 5] >> ((i + e) & 31) & 1) wt[e] = 0.0;
                            mine += wt[e];
                        }
                        double inc = mine;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const double y = __shfl_up_sync(0xffffffffu, inc, o);
                            if (lane >= o) inc += y;
                        }
                        double c = run + (inc - mine);
                        uint32_t hit = ~0u, pos = ~0u;
#pragma unroll
                        for (int e = 0; e < E; e++) {
                            c += wt[e];
                            if (wt[e] > 0.0) {
                                pos = i + e;
                                if (hit == ~0u && c > goal) hit = i + e;
                            }
                        }
                        found = __reduce_min_sync(0xffffffffu, hit);
                        const uint32_t any = __ballot_sync(0xffffffffu, pos != ~0u);
                        if (any) some = __shfl_sync(0xffffffffu, pos, 31 - __clz(any));
                        run += __shfl_sync(0xffffffffu, inc, 31);
                    }
                    if (lane == 0) a.next[r] = (int32_t)(found != ~0u ? found : some);
                }
            }
            answer = who < ctas ? -2 : -1;  // (written by that CTA)
            break;
        }
        if (rank == 0) {
            if (tid == 0) {
                a.accepted[r] = (int32_t)length;
                if (answer != -2) a.next[r] = answer;
            }
            for (uint32_t i = length + tid; i < most; i += THREADS) a.path[(size_t)r * most + i] = -1;
        }
        cluster_sync();  // the request's nodes have been read by all
    }
}

}  // namespace pv

template <int SRC, bool VEC> static cudaError_t verify_launch(const PagedVerifyArgs &a, uint32_t ctas, int sm_count, bool pdl, cudaStream_t stream) {
    auto *kernel = pv::paged_verify_kernel<SRC, VEC>;
    constexpr uint32_t E = SRC == ACT_F32 ? 4 : 8, unit = 32 * E;
    const uint32_t warps = ctas * pv::WARPS, part = ((a.vocab + warps - 1) / warps + unit - 1) / unit * unit;
    const size_t smem = pv::shared_bytes(a.s.max_new, part);
    static std::once_flag once[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    std::call_once(once[dev & 63], [&] { e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pv::shared_bytes(PAGED_TREE_MOST, PAGED_VERIFY_VOCAB / pv::WARPS / pv::MOST_CTAS)); });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    const uint32_t clusters = std::min<uint32_t>(a.s.requests, std::max<uint32_t>(1, 2 * (uint32_t)sm_count / ctas));
    cfg.gridDim = dim3(clusters * ctas);
    cfg.blockDim = dim3(pv::THREADS);
    cfg.dynamicSmemBytes = smem;
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
    const uint32_t eb = act_elem_bytes(a.type);
    const bool vec = (uintptr_t)a.logits % 16 == 0 && a.logits_row * eb % 16 == 0 && (!a.draft || ((uintptr_t)a.draft % 16 == 0 && a.draft_row % 4 == 0));
    const uint32_t ctas = pv::MOST_CTAS;
    auto run = [&](auto src) {
        constexpr int S = decltype(src)::value;
        return vec ? verify_launch<S, true>(a, ctas, sm_count, pdl, stream) : verify_launch<S, false>(a, ctas, sm_count, pdl, stream);
    };
    return a.type == ACT_F32 ? run(std::integral_constant<int, ACT_F32>()) : a.type == ACT_F16 ? run(std::integral_constant<int, ACT_F16>()) : run(std::integral_constant<int, ACT_BF16>());
}

}  // namespace lb
