// Attention of the new tokens of every request over its pages, the form that is simplest: a warp for each (token, query head) walks the keys
// with the running maximum m, sum l and accumulator of the softmax; a lane holds four elements of the head.
#include <cuda_bf16.h>

#include "common.cuh"
#include "paged.cuh"

namespace lb {

__device__ __forceinline__ float4 load_half4(const void *row, uint32_t i, bool bf16) {
    const uint2 w = *(const uint2 *)((const unsigned short *)row + i);
    const int t = bf16 ? ACT_BF16 : ACT_F16;
    return make_float4(widen_act(w.x & 0xffff, t), widen_act(w.x >> 16, t), widen_act(w.y & 0xffff, t), widen_act(w.y >> 16, t));
}

__global__ void __launch_bounds__(256) paged_attn_simple_kernel(PagedAttnArgs p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const PagedShape &s = p.s;
    if (p.plan[PLAN_STAMP] != p.stamp) {
        if (threadIdx.x == 0 && blockIdx.x == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_PLAN);
        return;
    }
    const uint32_t lane = threadIdx.x & 31, tokens = p.plan[PLAN_TOKENS];
    const bool has = 4 * lane < s.d;
    for (uint64_t w = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < (uint64_t)tokens * s.hq; w += (uint64_t)gridDim.x * 8) {
        const uint32_t t = (uint32_t)(w / s.hq), h = (uint32_t)(w % s.hq), kvh = h / s.g;
        uint32_t r = 0, top = s.requests;
        while (top - r > 1) {
            const uint32_t mid = (r + top) >> 1;
            if (p.plan[p.l.q_start + mid] <= t) r = mid;
            else top = mid;
        }
        const uint32_t q0 = p.plan[p.l.q_start + r], n = p.plan[p.l.q_start + r + 1] - q0, kv = p.plan[p.l.kv_len + r];
        const uint32_t hi = paged_hi(s, n, kv, t - q0), lo = paged_lo(s, hi);
        const unsigned short *qrow = (const unsigned short *)p.q + p.qv.off + (uint64_t)t * p.qv.token + (uint64_t)h * p.qv.head;
        const int at = s.bf16 ? ACT_BF16 : ACT_F16;
        float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o = q;
        if (has) q = make_float4(load_act(qrow, 4 * lane, at), load_act(qrow, 4 * lane + 1, at), load_act(qrow, 4 * lane + 2, at), load_act(qrow, 4 * lane + 3, at));
        float m = -INFINITY, l = 0.0f;
        bool bad = false;
        for (uint32_t j = lo; j < hi; j++) {
            const int32_t page = p.table[(size_t)r * s.max_blocks + j / s.page];
            const bool ok = page >= 0 && (uint32_t)page < s.pages;
            bad |= !ok;
            const size_t at_row = (((size_t)(ok ? page : 0) * s.hkv + kvh) * s.page + j % s.page) * s.d;
            float4 k = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = k;
            if (ok && has) k = load_half4((const unsigned short *)p.k_cache + at_row, 4 * lane, s.bf16), v = load_half4((const unsigned short *)p.v_cache + at_row, 4 * lane, s.bf16);
            float x = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, q.w * k.w)));
#pragma unroll
            for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            x *= s.scale;
            const float top_m = fmaxf(m, x), base = top_m == -INFINITY ? 0.0f : top_m, keep = expf(m - base), e = expf(x - base);
            m = top_m;
            l = fmaf(l, keep, e);
            o = make_float4(fmaf(o.x, keep, e * v.x), fmaf(o.y, keep, e * v.y), fmaf(o.z, keep, e * v.z), fmaf(o.w, keep, e * v.w));
        }
        if (bad && lane == 0 && p.status) atomicOr(p.status, (int)PAGED_STATUS_INDEX);
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        unsigned short *orow = (unsigned short *)p.out + p.ov.off + (uint64_t)t * p.ov.token + (uint64_t)h * p.ov.head;
        if (has) {
            const float f[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
            for (int i = 0; i < 4; i++) {
                if (s.bf16) ((__nv_bfloat16 *)orow)[4 * lane + i] = __float2bfloat16_rn(f[i]);
                else ((__half *)orow)[4 * lane + i] = __float2half_rn(f[i]);
            }
        }
        if (p.lse && lane == 0) p.lse[(size_t)t * s.hq + h] = l > 0.0f || l != l ? m + logf(l) : -INFINITY;
    }
}

uint32_t paged_attn_small_ctas(int sm_count) { return (uint32_t)sm_count; }
uint32_t paged_attn_large_ctas(int sm_count) { return (uint32_t)sm_count; }

cudaError_t launch_paged_attn_small(const PagedAttnArgs &a, int sm_count, bool pdl, cudaStream_t stream) {
    const uint64_t warps = (uint64_t)a.s.tokens * a.s.hq, want = (warps + 7) / 8, cap = (uint64_t)sm_count * 64;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)(want < cap ? want : cap));
    cfg.blockDim = dim3(256);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, paged_attn_simple_kernel, a);
}
cudaError_t launch_paged_attn_large(const PagedAttnArgs &, int, bool, cudaStream_t) { return cudaSuccess; }

}  // namespace lb
