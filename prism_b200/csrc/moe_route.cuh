// A token's choice of experts from its router's logits, and what an expert does between its products.
#pragma once

#include "common.cuh"

namespace prism {

__device__ __forceinline__ float moe_sigmoid(float z) { return 1.f / (1.f + expf(-z)); }
__device__ __forceinline__ float moe_act(float z, int act) {
    if (act == 0) return z / (1.f + expf(-z));                                                      // silu
    if (act == 1) return 0.5f * z * (1.f + tanhf(0.7978845608028654f * (z + 0.044715f * z * z * z)));   // gelu_tanh
    const float r = fmaxf(z, 0.f);
    return act == 3 ? r * r : r;                                                                      // relu squared, relu
}

// an expert's hidden value from its gate and up values; act 4: the clamped form (common.cuh: clamped_glu)
__device__ __forceinline__ float moe_glu(float g, float u, int act, float limit) {
    return act == 4 ? clamped_glu(g, u, limit) : moe_act(g, act) * u;
}

// One warp takes a token: scores into s [E] (shared), choice scores into c [E] (the score plus a correction per expert,
// where one is given), the `top` largest choice scores chosen (the lower index wins a tie), counts [E] (shared or global)
// raised by one per choice, whose old value is the choice's rank among its expert's rows.  With `groups` > 1 the experts
// form that many equal groups of neighbours, a group's score is its largest choice score, and only the experts of the
// best `keep` groups can be chosen (gs: 2 groups floats of scratch).  A choice's weight is its score without the
// correction, with renorm divided by the sum of the chosen (+ sum_eps), times wscale.
__device__ __forceinline__ void moe_route_token(const float* __restrict__ z, float* s, float* c, float* gs, int E, int top,
                                                int softmax, int renorm, int lane, int* counts, int* __restrict__ sel_e,
                                                float* __restrict__ sel_w, int* __restrict__ sel_rank,
                                                const void* __restrict__ corr, int corr_bf16, int groups, int keep,
                                                float wscale, float sum_eps) {
    float mx = -INFINITY;
    for (int e = lane; e < E; e += 32) mx = fmaxf(mx, z[e]);
    mx = warp_max(mx);
    float den = 0.f;
    for (int e = lane; e < E; e += 32) {
        const float v = softmax ? expf(z[e] - mx) : moe_sigmoid(z[e]);
        s[e] = v;
        den += v;
    }
    den = warp_sum(den);
    __syncwarp();
    for (int e = lane; e < E; e += 32) {
        const float v = softmax ? s[e] / den : s[e];
        s[e] = v;
        c[e] = corr != nullptr ? v + load_param(corr, corr_bf16, e) : v;
    }
    __syncwarp();
    if (groups > 1 && keep < groups) {
        const int per = E / groups;
        float* kept = gs + groups;
        for (int g = lane; g < groups; g += 32) {
            float best = -INFINITY;
            for (int e = g * per; e < (g + 1) * per; ++e) best = fmaxf(best, c[e]);
            gs[g] = best;
            kept[g] = 0.f;
        }
        __syncwarp();
        for (int j = 0; j < keep; ++j) {
            float best = -INFINITY;
            int at = groups;
            for (int g = lane; g < groups; g += 32)
                if (kept[g] == 0.f && (gs[g] > best || at == groups)) { best = gs[g]; at = g; }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float ob = __shfl_xor_sync(0xffffffffu, best, o);
                const int oa = __shfl_xor_sync(0xffffffffu, at, o);
                if (oa < groups && (at == groups || ob > best || (ob == best && oa < at))) { best = ob; at = oa; }
            }
            if (lane == 0 && at < groups) kept[at] = 1.f;
            __syncwarp();
        }
        for (int e = lane; e < E; e += 32)
            if (kept[e / per] == 0.f) c[e] = -INFINITY;
        __syncwarp();
    }
    float chosen = 0.f;
    for (int j = 0; j < top; ++j) {
        float best = -INFINITY;
        int at = E;
        for (int e = lane; e < E; e += 32)
            if (c[e] > best) { best = c[e]; at = e; }           // ascending e: the lowest index of equal scores
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ob = __shfl_xor_sync(0xffffffffu, best, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
        }
        if (at >= E) at = 0;                                   // every score NaN: keep the indices legal
        const float w = s[at];
        chosen += w;
        if (lane == 0) {
            sel_e[j] = at;
            sel_w[j] = w;
            sel_rank[j] = atomicAdd(counts + at, 1);
            c[at] = -INFINITY;
        }
        __syncwarp();
    }
    if (lane == 0)
        for (int j = 0; j < top; ++j) sel_w[j] = (renorm ? sel_w[j] / (chosen + sum_eps) : sel_w[j]) * wscale;
}

}  // namespace prism
