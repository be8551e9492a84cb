// The routed experts' choice for one token, shared by the kernels that make it.
#pragma once

#include "common.cuh"

// ---------------------------------------------------------------------------------------------------------------
// the router's choice: one warp per token
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void warp_argmax(float& v, int& i) {      // the largest value, the lowest index among equals
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, v, o);
        const int oi = __shfl_xor_sync(0xffffffffu, i, o);
        if (ov > v || (ov == v && oi < i)) {
            v = ov;
            i = oi;
        }
    }
}

// One warp: the choice for one token from its E logits `zr`; scratch: 2 E + 2 groups floats of the warp's own.
// scoring 0: s = softmax(z); 1: s = sigmoid(z).  renorm: the chosen weights are divided by their sum; then all are multiplied by wscale.
// The choice goes by c = s + correction (null: c = s), which may be negative; a run of experts is scored by its best c, or
// with pair_sum by the sum of its two best (a run of one: its only one).
__device__ __forceinline__ void moe_route_warp(const float* zr, float* scratch, int lane, int E, int top, int groups, int keep,
                                               int32_t* __restrict__ idx, float* __restrict__ wts, size_t t, int scoring = 0,
                                               const float* __restrict__ correction = nullptr, int pair_sum = 0, int renorm = 1, float wscale = 1.0f) {
    float* s = scratch;
    float* c = scratch + E;
    float* gs = scratch + 2 * E;
    float* kept = gs + groups;
    if (scoring == 1) {
        for (int e = lane; e < E; e += 32) s[e] = 1.0f / (1.0f + expf(-zr[e]));
    } else {
        float m = -INFINITY;
        for (int e = lane; e < E; e += 32) m = fmaxf(m, zr[e]);
        m = warp_max(m);
        float sum = 0.0f;
        for (int e = lane; e < E; e += 32) {
            const float p = expf(zr[e] - m);
            s[e] = p;
            sum += p;
        }
        sum = warp_sum(sum);
        const float inv = 1.0f / sum;
        for (int e = lane; e < E; e += 32) s[e] *= inv;
    }
    for (int e = lane; e < E; e += 32) c[e] = correction ? s[e] + correction[e] : s[e];
    __syncwarp();
    const int size = E / groups;
    if (keep < groups) {
        for (int g = lane; g < groups; g += 32) {
            float b = -INFINITY, b2 = -INFINITY;
            for (int e = 0; e < size; ++e) {
                const float v = c[g * size + e];
                if (v > b) {
                    b2 = b;
                    b = v;
                } else {
                    b2 = fmaxf(b2, v);
                }
            }
            gs[g] = pair_sum && size > 1 ? b + b2 : b;
        }
        __syncwarp();
        // a run stays when fewer than `keep` runs are ahead of it (a better score, or an equal one and a lower index)
        for (int g = lane; g < groups; g += 32) {
            int ahead = 0;
            for (int o = 0; o < groups; ++o) ahead += gs[o] > gs[g] || (gs[o] == gs[g] && o < g);
            kept[g] = ahead < keep ? 1.0f : 0.0f;
        }
        __syncwarp();
        for (int e = lane; e < E; e += 32)
            if (kept[e / size] == 0.0f) c[e] = -INFINITY;      // not eligible
        __syncwarp();
    }
    float total = 0.0f;
    for (int kk = 0; kk < top; ++kk) {
        float bv = -INFINITY;
        int bi = 0x7fffffff;
        for (int e = lane; e < E; e += 32)
            if (c[e] > bv) {
                bv = c[e];
                bi = e;
            }
        warp_argmax(bv, bi);
        float weight = 0.0f;
        if (bi == 0x7fffffff) {     // fewer eligible experts than `top`: the rest of the choice carries no weight
            bi = 0;
        } else {
            weight = s[bi];
            if (lane == 0) c[bi] = -INFINITY;
        }
        __syncwarp();
        total += weight;
        if (lane == 0) {
            idx[t * top + kk] = bi;
            wts[t * top + kk] = weight;
        }
    }
    __syncwarp();
    if (lane == 0 && (renorm || wscale != 1.0f)) {
        const float d = renorm ? total + 1e-20f : 1.0f;
        for (int kk = 0; kk < top; ++kk) wts[t * top + kk] = wts[t * top + kk] / d * wscale;
    }
}
