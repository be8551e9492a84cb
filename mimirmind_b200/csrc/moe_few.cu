// A whole routed-experts layer for up to 16 tokens in two launches.
//
//   z = x W_router^T;  the choice of `top` experts and their weights (moe_route.cuh)
//   h[t, c] = act(W_gate[e] x_t, W_up[e] x_t),   out[t] = sum over the choices c in order of wts[t, c] W_down[e] h[t, c],   e = idx[t, c].
//
// A few tokens are bound by the chosen experts' matrices: each is read once, by mma.sync with 16 weight rows as the 16-row operand and the expert's
// rows of x, found by their places, as its 8 (or twice 8) columns.  Nothing is sorted or copied.
//
// First launch, clusters of eight CTAs: every cluster makes all logits (an eighth of the router's rows each, handed round over distributed
// shared memory), every CTA makes the choice and the list of experts with their tokens; then its share of the units of 8 gate and 8 up rows.
// That costs a read of the router per cluster from L2 and saves a launch and its wait for another.
// Second launch: 16 output columns a CTA; its warps share out the experts' runs of hidden columns, whose sums are kept apart per (token, choice) and added
// in the order of the choice.  A token's output does not depend on the others: every sum is cut by the layer's sizes alone.
//
// The router's weights are fp32: each is three bf16 parts (hi, mid, lo, 24 bits together), x is bf16, the sums are fp32.
// Experts in bf16: x as it is, the fp32 hidden rows as two bf16 parts (2^-17 of a number is lost).  Experts in e4m3 with a scale per block of 128 x 128: weights
// become fp16 exactly; the rows of x and the hidden rows become fp16 after a power of two that brings their largest number to 2^14 .. 2^15
// (x loses nothing above 2^-29 of its largest, hidden rows keep 11 bits: rounding them to bf16 would cost as much again as rounding the result).
//
// Bound by memory: PLACEHOLDER
#include <cuda_fp16.h>

#include "fp8.cuh"
#include "fp8_launch.h"
#include "moe_route.cuh"

namespace {

constexpr int FEW_THREADS = 512, FEW_WARPS = 16, FEW_RING = 3, FEW_SLOT = 2048, FEW_CLUSTER = 8;
constexpr int FEW_TOKENS = 16, FEW_MAX_EXPERTS = 512, FEW_MAX_TOP = 32;
constexpr int FEW_CLUSTERS = FP8_SM_COUNT / FEW_CLUSTER;      // at the most

struct FewArgs {
    const __nv_bfloat16* x;
    const float* w_router;
    const float* correction;
    const uint8_t *w_in, *w_out;          // rows of ld_in, ld_out bytes
    const float *s_in, *s_out;            // e4m3: scales
    float* hidden;                        // [pairs][F]
    uint32_t* largest;                    // [pairs][F / 8]: bits of the units' largest sizes
    int32_t* lists;                       // entries' number, entries (expert, first place, rows) 3 each, places' pairs
    float* weights;                       // [pairs]
    uint16_t* x_half;                     // e4m3 experts: [clusters][n][D] fp16
    __nv_bfloat16* out;
    long long ldx, ld_in, ld_out;
    int n, D, E, top, groups, keep, scoring, renorm, pair_sum, F, act, on_input, interleaved;
    float wscale, limit;
    int KS, splits;
};

__device__ __forceinline__ void few_copy16(uint32_t dst, const uint8_t* row, int at, int bytes) {      // 16 bytes of a row, noughts behind its end
    const int n = min(max(bytes - at, 0), 16);
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(n > 0 ? row + at : row), "r"(n) : "memory");
}
__device__ __forceinline__ void few_copy16(uint32_t dst, const uint8_t* src) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void few_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

__device__ __forceinline__ void mma_bf16_f32(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_f32(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float low_of(uint32_t bf16_pair) { return __uint_as_float(bf16_pair << 16); }
__device__ __forceinline__ float high_of(uint32_t bf16_pair) { return __uint_as_float(bf16_pair & 0xffff0000u); }
// four e4m3 numbers as two fp16 pairs
__device__ __forceinline__ void f16_of(uint32_t w, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(a), "=r"(b) : "r"(w));
}

// The power of two that brings a size to 2^14 .. 2^15 (sizes below 2^-112: 2^126), and its inverse; an infinity or a NaN stays one under it.
__device__ __forceinline__ float f16_scale(uint32_t size_bits) {
    const int e = min(max((int)(size_bits >> 23), 15), 254);
    return __uint_as_float((uint32_t)(268 - e) << 23);
}
__device__ __forceinline__ float f16_unscale(uint32_t size_bits) {
    const int e = min(max((int)(size_bits >> 23), 15), 254);
    return __uint_as_float((uint32_t)(e - 14) << 23);
}

// moe_route_warp's choice where every run of experts is kept: a choice is two reductions over the warp.  Code that runs once in a launch is
// fetched from L2 as it goes: kept short, it takes 2,000 cycles for 8 of 128 experts instead of 7,600.
// s: 2 E words of the warp's own: the scores, and their order (0: not to be chosen, a NaN, minus infinity or chosen already).
__device__ __forceinline__ void few_choose(const float* __restrict__ z, float* s, int lane, int E, int top, int scoring, const float* __restrict__ correction, int renorm,
                                           float wscale, int32_t* idx, float* wts) {
    uint32_t* key = reinterpret_cast<uint32_t*>(s + E);
    float m = 0.0f, inv = 1.0f;
    if (scoring == 0) {
        m = -INFINITY;
#pragma unroll 1
        for (int e = lane; e < E; e += 32) m = fmaxf(m, z[e]);
        m = warp_max(m);
        float sum = 0.0f;
#pragma unroll 1
        for (int e = lane; e < E; e += 32) {
            const float p = expf(z[e] - m);
            s[e] = p;
            sum += p;
        }
        inv = 1.0f / warp_sum(sum);
    }
#pragma unroll 1
    for (int e = lane; e < E; e += 32) {
        const float v = scoring == 1 ? 1.0f / (1.0f + expf(-z[e])) : s[e] * inv;
        s[e] = v;
        const float c = correction ? v + correction[e] : v;
        const uint32_t u = __float_as_uint(c);
        key[e] = c != c || c == -INFINITY ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
    }
    __syncwarp();
    float total = 0.0f, mine_w = 0.0f;
    int mine_e = 0;
#pragma unroll 1
    for (int k = 0; k < top; ++k) {
        uint32_t best = 0;
        int at = 0x7fffffff;
#pragma unroll 1
        for (int e = lane; e < E; e += 32) {
            const uint32_t v = key[e];
            if (v > best) {
                best = v;
                at = e;
            }
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        int e = (int)__reduce_min_sync(0xffffffffu, best == most && most != 0 ? (uint32_t)at : 0x7fffffffu);      // the lowest number among equals
        float weight = 0.0f;
        if (e == 0x7fffffff) {
            e = 0;               // fewer to choose from than `top`: the rest of the choice carries no weight
        } else {
            weight = s[e];
            if ((e & 31) == lane) key[e] = 0;
        }
        __syncwarp();
        total += weight;
        if (lane == k) {
            mine_e = e;
            mine_w = weight;
        }
    }
    if (lane < top) {
        idx[lane] = mine_e;
        wts[lane] = renorm || wscale != 1.0f ? mine_w / (renorm ? total + 1e-20f : 1.0f) * wscale : mine_w;
    }
}

// A slot of a warp's ring: 128 bytes of 16 weight rows (a lane's four pieces: bytes t * 16 .. + 15 and 64 on of rows g and g + 8), 128 e4m3 or 64
// bf16 numbers a row.  The order of k inside it is free as long as both operands agree: a lane's pieces are multiplied as they lie.

// numbers of a row of x in shared memory: rows of neighbouring columns lie in different banks (a lane takes 32 bytes beside e4m3 weights, 16 beside bf16)
__host__ __device__ inline int few_x_stride(int D, bool fp8) { return (D + 63) / 64 * 64 + (fp8 ? 8 : 32); }
// 4-byte words in front of the rows that make them start on 16 bytes
__host__ __device__ inline int few_pad(int n, int E, int pairs) { return (-(((n * E + 3) & ~3) + 6 * pairs + 2 * FEW_WARPS + 2 + FEW_TOKENS)) & 3; }

// ---------------------------------------------------------------------------------------------------------------
// first launch: router, choice, gate and up products, activation
// ---------------------------------------------------------------------------------------------------------------
template <bool FP8, int G, bool XS>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_in_kernel(const __grid_constant__ FewArgs g) {
    constexpr int TOK = 8 * G;
    extern __shared__ __align__(16) unsigned char few_smem[];
    unsigned char* rings = few_smem;                                                            // later also the choice's scratch
    float* part = reinterpret_cast<float*>(few_smem + FEW_WARPS * FEW_RING * FEW_SLOT);         // [2][16 warps][16][TOK]
    float* logits = part + 2 * FEW_WARPS * 16 * TOK;                                            // [n][E]
    const int pairs = g.n * g.top;
    int32_t* idx = reinterpret_cast<int32_t*>(logits + ((g.n * g.E + 3) & ~3));                // [pairs]
    float* wts = reinterpret_cast<float*>(idx + pairs);                                         // [pairs]
    int32_t* places = reinterpret_cast<int32_t*>(wts + pairs);                                  // [pairs]: the pair at every place, by expert
    int32_t* entries = places + pairs;                                                          // [pairs][3]
    int32_t* sums = entries + 3 * pairs;                                                        // [2][16 warps], [2] totals
    uint32_t* x_largest = reinterpret_cast<uint32_t*>(sums + 2 * FEW_WARPS + 2);                // [16]
    uint16_t* x_rows = reinterpret_cast<uint16_t*>(x_largest + FEW_TOKENS + few_pad(g.n, g.E, pairs));      // XS: [n][x_stride]
    const int x_stride = few_x_stride(g.D, FP8);
    uint16_t* x_half = FP8 && !XS ? g.x_half + (size_t)(blockIdx.x / FEW_CLUSTER) * g.n * g.D : nullptr;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t4 = lane & 3;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    pdl_trigger();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // waited for in front of the first store to another CTA: by then it runs

    if (FP8) {
        if (warp < g.n) {            // a warp per token
            uint32_t big = 0;
#pragma unroll 4
            for (int d = lane * 8; d < g.D; d += 256) {       // (D is a multiple of 8)
                const uint4 v = *reinterpret_cast<const uint4*>(g.x + (size_t)warp * g.ldx + d);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) big = max(big, max((w[i] & 0x7fffu) << 16, w[i] & 0x7fff0000u));
            }
            big = __reduce_max_sync(0xffffffffu, big);
            if (lane == 0) x_largest[warp] = big;
        }
        __syncthreads();
    }
    // x as the products read it: into shared memory, or (rows too long for that; e4m3 experts) the cluster's own copy in memory, an eighth by every CTA
    // (read behind the cluster's barrier)
    if (XS || FP8) {
        const int chunks = g.D / 8, first = XS ? threadIdx.x : rank * FEW_THREADS + threadIdx.x, step = XS ? FEW_THREADS : FEW_CLUSTER * FEW_THREADS;
#pragma unroll 4
        for (int i = first; i < g.n * chunks; i += step) {
            const int t = i / chunks, d = (i - t * chunks) * 8;
            uint4 v = *reinterpret_cast<const uint4*>(g.x + (size_t)t * g.ldx + d);
            if (FP8) {
                const float s = f16_scale(x_largest[t]);
                v = make_uint4(pair_f16(low_of(v.x) * s, high_of(v.x) * s), pair_f16(low_of(v.y) * s, high_of(v.y) * s), pair_f16(low_of(v.z) * s, high_of(v.z) * s),
                               pair_f16(low_of(v.w) * s, high_of(v.w) * s));
            }
            *reinterpret_cast<uint4*>(XS ? x_rows + (size_t)t * x_stride + d : x_half + (size_t)t * g.D + d) = v;
        }
    }
    // ---- logits: 16 experts a tile, a sixteenth of the depth a warp ----
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    {
        const int steps = (g.D + 15) / 16, lo = steps * warp / FEW_WARPS, hi = steps * (warp + 1) / FEW_WARPS;
        for (int tile = rank; tile * 16 < g.E; tile += FEW_CLUSTER) {
            const float *wa = g.w_router + (size_t)min(tile * 16 + gr, g.E - 1) * g.D, *wb = g.w_router + (size_t)min(tile * 16 + gr + 8, g.E - 1) * g.D;
            float acc[G][4];
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
#pragma unroll (G == 1 ? 4 : 2)
            for (int s = lo; s < hi; ++s) {
                const int k = s * 16 + t4 * 4;
                const bool on = k < g.D;
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float4 a = on ? *reinterpret_cast<const float4*>(wa + k) : zero, b = on ? *reinterpret_cast<const float4*>(wb + k) : zero;
                uint2 xv[G];
#pragma unroll
                for (int j = 0; j < G; ++j)
                    xv[j] = on && j * 8 + gr < g.n ? *reinterpret_cast<const uint2*>(g.x + (size_t)(j * 8 + gr) * g.ldx + k) : make_uint2(0, 0);
                float r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int p = 0; p < 3; ++p) {       // hi, mid, lo
                    const uint32_t a0 = pair_bf16(r[0], r[1]), a2 = pair_bf16(r[2], r[3]), a1 = pair_bf16(r[4], r[5]), a3 = pair_bf16(r[6], r[7]);
                    if (p < 2) {
                        r[0] -= low_of(a0); r[1] -= high_of(a0); r[2] -= low_of(a2); r[3] -= high_of(a2);
                        r[4] -= low_of(a1); r[5] -= high_of(a1); r[6] -= low_of(a3); r[7] -= high_of(a3);
                    }
#pragma unroll
                    for (int j = 0; j < G; ++j) mma_bf16_f32(acc[j], a0, a1, a2, a3, xv[j].x, xv[j].y);
                }
            }
            float* mine = part + (warp * 16 + gr) * TOK + t4 * 2;
            __syncthreads();        // the tile before has been read
#pragma unroll
            for (int j = 0; j < G; ++j) {
                *reinterpret_cast<float2*>(mine + j * 8) = make_float2(acc[j][0], acc[j][1]);
                *reinterpret_cast<float2*>(mine + 8 * TOK + j * 8) = make_float2(acc[j][2], acc[j][3]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * g.n; i += FEW_THREADS) {
                const int row = i & 15, tok = i >> 4, e = tile * 16 + row;
                float z = 0.0f;
#pragma unroll
                for (int w = 0; w < FEW_WARPS; ++w) z += part[(w * 16 + row) * TOK + tok];
                if (e < g.E) {
                    const uint32_t at = (uint32_t)__cvta_generic_to_shared(logits + tok * g.E + e);
#pragma unroll
                    for (int r = 0; r < FEW_CLUSTER; ++r) {
                        uint32_t there;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(r));
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(z) : "memory");
                    }
                }
            }
        }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (no CTA has more logits to hand out behind this: one barrier does)
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

    // ---- the choice: a warp per token ----
    if (warp < g.n && g.keep == g.groups)
        few_choose(logits + warp * g.E, reinterpret_cast<float*>(rings) + (size_t)warp * 2 * g.E, lane, g.E, g.top, g.scoring, g.correction, g.renorm, g.wscale,
                   idx + warp * g.top, wts + warp * g.top);
    else if (warp < g.n)
        moe_route_warp(logits + warp * g.E, reinterpret_cast<float*>(rings) + (size_t)warp * 2 * (g.E + g.groups), lane, g.E, g.top, g.groups, g.keep, idx, wts,
                       (size_t)warp, g.scoring, g.correction, g.pair_sum, g.renorm, g.wscale);
    __syncthreads();
    // ---- the experts that someone chose, in order, with their pairs (token * top + choice): a thread per expert ----
    {
        const int e = threadIdx.x;
        int count = 0;
        if (e < g.E) {
            int p = 0;
            for (; p + 4 <= pairs; p += 4) {
                const int4 v = *reinterpret_cast<const int4*>(idx + p);
                count += (v.x == e) + (v.y == e) + (v.z == e) + (v.w == e);
            }
            for (; p < pairs; ++p) count += idx[p] == e;
        }
        const int parts = (count + TOK - 1) / TOK;
        int upto = count, parts_upto = parts;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, upto, o), b = __shfl_up_sync(0xffffffffu, parts_upto, o);
            if (lane >= o) {
                upto += a;
                parts_upto += b;
            }
        }
        if (lane == 31) {
            sums[warp] = upto;
            sums[FEW_WARPS + warp] = parts_upto;
        }
        __syncthreads();
        int first = upto - count, entry = parts_upto - parts;
        for (int w = 0; w < warp; ++w) {
            first += sums[w];
            entry += sums[FEW_WARPS + w];
        }
        if (threadIdx.x == FEW_THREADS - 1) sums[2 * FEW_WARPS] = entry + parts;
        if (count > 0) {
            int at = first;
            for (int p = 0; p < pairs; ++p)
                if (idx[p] == e) places[at++] = p;
            for (int i = 0; i < parts; ++i) {
                entries[3 * (entry + i)] = e;
                entries[3 * (entry + i) + 1] = first + i * TOK;
                entries[3 * (entry + i) + 2] = min(TOK, count - i * TOK);
            }
        }
        __syncthreads();
    }
    const int n_entries = sums[2 * FEW_WARPS];
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) g.lists[0] = n_entries;
        for (int i = threadIdx.x; i < 3 * n_entries; i += FEW_THREADS) g.lists[1 + i] = entries[i];
        for (int i = threadIdx.x; i < pairs; i += FEW_THREADS) {
            g.lists[1 + 3 * pairs + i] = places[i];
            g.weights[i] = g.on_input ? 1.0f : wts[i];
        }
    }

    // ---- units of 8 gate and 8 up rows, a unit's depth in KS runs: a warp per run and the runs' sums added over shared memory, or, where there are many
    // units, a warp per unit that goes through the runs itself.  The sums are the same to the bit.  The cheaper one by rounds of slots (a meeting of the
    // warps costs about two)  ----
    constexpr int PER = FP8 ? 128 : 64;                  // numbers in a slot's row
    const int bytes = FP8 ? g.D : 2 * g.D, blocks = (bytes + 127) / 128, uf = g.F / 8, units = n_entries * uf;
    const int side = FEW_WARPS / g.KS;
    const bool alone = (units + (int)gridDim.x * FEW_WARPS - 1) / ((int)gridDim.x * FEW_WARPS) * blocks <=
                       (units + (int)gridDim.x * side - 1) / ((int)gridDim.x * side) * (blocks / g.KS + 2);
    const int RT = alone ? FEW_WARPS : side, rt = alone ? warp : warp / g.KS, run_lo = alone ? 0 : warp % g.KS, run_hi = alone ? g.KS : run_lo + 1;
    const int lo = blocks * run_lo / g.KS, hi = blocks * run_hi / g.KS, nb = hi - lo;
    const int groups = (units + RT - 1) / RT, steps = (int)blockIdx.x < groups ? (groups - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    // (warps that are alone take every grid's-width unit, so that few units are spread over all CTAs)
    const int stride = (int)gridDim.x * RT, unit0 = alone ? (int)blockIdx.x + rt * (int)gridDim.x : (int)blockIdx.x * RT + rt;
    const int my_steps = alone ? (unit0 < units ? (units - 1 - unit0) / stride + 1 : 0) : steps;
    unsigned char* ring = rings + warp * FEW_RING * FEW_SLOT;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const int kb = (g.D + 127) / 128, fb = (g.F + 127) / 128;
    // a place in the units: (entry, unit of 8 columns), carried along; behind the last unit it stays on it (not stored)
    struct Cursor {
        int entry, fu;
    };
    auto cursor_at = [&](int u) {
        u = min(u, units - 1);
        return Cursor{u / uf, u % uf};
    };
    auto advance = [&](Cursor& c) {
        c.fu += stride;
        while (c.fu >= uf && c.entry < n_entries) {
            c.fu -= uf;
            ++c.entry;
        }
        if (c.entry >= n_entries) c = {n_entries - 1, uf - 1};
    };
    const uint8_t *pa = nullptr, *pb = nullptr;
    Cursor ahead = cursor_at(unit0), here = ahead;
    int load_b = lo;
    auto point = [&]() {
        const int e = entries[3 * ahead.entry], f = ahead.fu * 8 + gr;
        size_t ra, rb;
        if (!FP8 && g.interleaved) {
            ra = (size_t)2 * e * g.F + 2 * (f - gr) + gr;
            rb = ra + 8;
        } else {
            ra = (size_t)2 * e * g.F + f;
            rb = ra + g.F;
        }
        pa = g.w_in + ra * g.ld_in;
        pb = g.w_in + rb * g.ld_in;
    };
    const int total = nb * my_steps;
    const bool whole = bytes % 128 == 0;
    auto load = [&](int slot) {
        const uint32_t dst = ring_at + slot * FEW_SLOT;
        const int at = load_b * 128 + t4 * 16;
        if (whole) {
            few_copy16(dst, pa + at);
            few_copy16(dst + 512, pb + at);
            few_copy16(dst + 1024, pa + at + 64);
            few_copy16(dst + 1536, pb + at + 64);
        } else {
            few_copy16(dst, pa, at, bytes);
            few_copy16(dst + 512, pb, at, bytes);
            few_copy16(dst + 1024, pa, at + 64, bytes);
            few_copy16(dst + 1536, pb, at + 64, bytes);
        }
        if (++load_b == hi) {
            load_b = lo;
            advance(ahead);
            point();
        }
    };
    if (total > 0) point();
#pragma unroll 1
    for (int i = 0; i < FEW_RING; ++i) {
        if (i < total) load(i);
        few_commit();
    }
    int done = 0, slot = 0;
#pragma unroll 1
    for (int step = 0; step < my_steps; ++step) {
        const int first = entries[3 * here.entry + 1], count = entries[3 * here.entry + 2], f0 = here.fu * 8;
        const uint16_t* rows[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int t = places[first + min(j * 8 + gr, count - 1)] / g.top;
            rows[j] = (XS ? x_rows + t * x_stride : FP8 ? x_half + (size_t)t * g.D : reinterpret_cast<const uint16_t*>(g.x) + (size_t)t * g.ldx) + t4 * (PER / 8);
        }
        const float *sg = nullptr, *su = nullptr;
        if (FP8) {
            sg = g.s_in + ((size_t)2 * entries[3 * here.entry] * fb + f0 / 128) * kb;
            su = sg + (size_t)fb * kb;
        }
        float s0_next = FP8 ? sg[lo] : 1.0f, s1_next = FP8 ? su[lo] : 1.0f;
        float sum[G][4];
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[j][c] = 0.0f;
#pragma unroll 1
        for (int run = run_lo; run < run_hi; ++run) {
            float acc[G][4];
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
            const int end = blocks * (run + 1) / g.KS;
#pragma unroll 1
            for (int b = blocks * run / g.KS; b < end; ++b) {
                // the rows of x first: they come while the weights are waited for
                constexpr int XW = FP8 ? 2 : 1;              // 16-byte pieces of x beside 16 bytes of a weight row
                uint4 xv[G][2][XW];
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < XW; ++i) {
                            const int k = b * PER + h * (PER / 2) + i * 8;
                            xv[j][h][i] = j * 8 + gr < count && (whole || k + t4 * (PER / 8) < g.D) ? *reinterpret_cast<const uint4*>(rows[j] + k) : make_uint4(0, 0, 0, 0);      // (D is a multiple of 8)
                        }
                const float s0 = s0_next, s1 = s1_next;
                if (FP8 && b + 1 < hi) {
                    s0_next = sg[b + 1];
                    s1_next = su[b + 1];
                }
                asm volatile("cp.async.wait_group %0;" ::"n"(FEW_RING - 1) : "memory");
                const unsigned char* at = ring + slot * FEW_SLOT + lane * 16;
                float c[G][2][4];            // two chains of products: one's results are 23 cycles away
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) c[j][i >> 2][i & 3] = 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 wl = *reinterpret_cast<const uint4*>(at + 1024 * h), wh = *reinterpret_cast<const uint4*>(at + 512 + 1024 * h);
                    const uint32_t lw[4] = {wl.x, wl.y, wl.z, wl.w}, hw[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
                    for (int i = 0; i < (FP8 ? 4 : 2); ++i) {
                        uint32_t a0, a1, a2, a3;
                        if (FP8) {
                            f16_of(lw[i], a0, a2);
                            f16_of(hw[i], a1, a3);
                        } else {
                            a0 = lw[2 * i];
                            a2 = lw[2 * i + 1];
                            a1 = hw[2 * i];
                            a3 = hw[2 * i + 1];
                        }
#pragma unroll
                        for (int j = 0; j < G; ++j) {
                            if (j > 0 && count <= 8 * j) break;
                            const uint4 v = xv[j][h][FP8 ? i >> 1 : 0];
                            const uint32_t p0 = (i & 1) ? v.z : v.x, p1 = (i & 1) ? v.w : v.y;
                            if (FP8) mma_f16_f32(c[j][h], a0, a1, a2, a3, p0, p1);
                            else mma_bf16_f32(h ? c[j][1] : acc[j], a0, a1, a2, a3, p0, p1);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[j][i] = FP8 ? fmaf(i < 2 ? s0 : s1, c[j][0][i] + c[j][1][i], acc[j][i]) : acc[j][i] + c[j][1][i];
                if (done + FEW_RING < total) load(slot);
                few_commit();
                ++done;
                slot = slot + 1 == FEW_RING ? 0 : slot + 1;
            }
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[j][c] += acc[j][c];
        }
        if (alone) {
#pragma unroll
            for (int j = 0; j < G; ++j) {
                if (j > 0 && count <= 8 * j) break;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = j * 8 + t4 * 2 + c;
                    const bool on = col < count;
                    const int pair = on ? places[first + col] : 0;
                    float y = sum[j][c], v = sum[j][2 + c];
                    if (FP8) {
                        const float back = f16_unscale(x_largest[pair / g.top]);
                        y *= back;
                        v *= back;
                    }
                    const float h = fp8_glu(y, v, g.act, g.limit, g.on_input ? wts[pair] : 1.0f);
                    if (on) g.hidden[(size_t)pair * g.F + f0 + gr] = h;
                    if (FP8) {
                        uint32_t big = fp8_size_bits(h);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
                        if (on && gr == 0) g.largest[(size_t)pair * uf + f0 / 8] = big;
                    }
                }
            }
        } else {
            float* mine = part + (((step & 1) * FEW_WARPS + warp) * 16 + gr) * TOK + t4 * 2;
#pragma unroll
            for (int j = 0; j < G; ++j) {
                *reinterpret_cast<float2*>(mine + j * 8) = make_float2(sum[j][0], sum[j][1]);
                *reinterpret_cast<float2*>(mine + 8 * TOK + j * 8) = make_float2(sum[j][2], sum[j][3]);
            }
            __syncthreads();
            // eight columns of a pair by eight neighbouring threads; other warps every time
            const float* all = part + (step & 1) * FEW_WARPS * 16 * TOK;
            for (int i = (threadIdx.x + step * 128) & (FEW_THREADS - 1); i < RT * TOK * 8; i += FEW_THREADS) {      // (a multiple of 32)
                const int f = i & 7, j = (i >> 3) % TOK, tile = (i >> 3) / TOK, unit = (int)blockIdx.x * RT + step * stride + tile;
                const Cursor at = cursor_at(unit);
                const bool on = unit < units && j < entries[3 * at.entry + 2];
                float h = 0.0f;
                int pair = 0;
                if (on) {
                    pair = places[entries[3 * at.entry + 1] + j];
                    const float* p = all + (tile * g.KS * 16 + f) * TOK + j;
                    float y = 0.0f, v = 0.0f;
                    for (int s = 0; s < g.KS; ++s) {
                        y += p[s * 16 * TOK];
                        v += p[s * 16 * TOK + 8 * TOK];
                    }
                    if (FP8) {
                        const float back = f16_unscale(x_largest[pair / g.top]);
                        y *= back;
                        v *= back;
                    }
                    h = fp8_glu(y, v, g.act, g.limit, g.on_input ? wts[pair] : 1.0f);
                    g.hidden[(size_t)pair * g.F + at.fu * 8 + f] = h;
                }
                if (FP8) {
                    uint32_t big = fp8_size_bits(h);
#pragma unroll
                    for (int o = 4; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
                    if (on && f == 0) g.largest[(size_t)pair * uf + at.fu] = big;
                }
            }
        }
        advance(here);
    }
}

// ---------------------------------------------------------------------------------------------------------------
// second launch: down products and the weighted sum
// ---------------------------------------------------------------------------------------------------------------
template <bool FP8, int G>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_out_kernel(const __grid_constant__ FewArgs g) {
    extern __shared__ __align__(16) unsigned char few_smem[];
    const int pairs = g.n * g.top;
    float* sums = reinterpret_cast<float*>(few_smem + FEW_WARPS * FEW_RING * FEW_SLOT);         // [splits][pairs][16]
    float* wts = sums + (size_t)g.splits * pairs * 16;                                          // [pairs]
    uint32_t* largest = reinterpret_cast<uint32_t*>(wts + pairs);                               // [pairs]
    int32_t* places = reinterpret_cast<int32_t*>(largest + pairs);                              // [pairs]
    int32_t* entries = places + pairs;                                                          // [pairs][3]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t4 = lane & 3;
    pdl_wait();
    const int n_entries = g.lists[0];
    for (int i = threadIdx.x; i < 3 * pairs; i += FEW_THREADS) entries[i] = g.lists[1 + i];       // (behind the entries: not read)
    for (int i = threadIdx.x; i < pairs; i += FEW_THREADS) {
        places[i] = g.lists[1 + 3 * pairs + i];
        wts[i] = g.weights[i];
    }
    __syncthreads();
    constexpr int PER = FP8 ? 128 : 64;
    const int bytes = FP8 ? g.F : 2 * g.F, blocks = (bytes + 127) / 128, items = n_entries * g.splits, n0 = blockIdx.x * 16;
    const int fb = (g.F + 127) / 128, db = (g.D + 127) / 128;
    unsigned char* ring = few_smem + warp * FEW_RING * FEW_SLOT;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const int ra = min(n0 + gr, g.D - 1), rb = min(n0 + gr + 8, g.D - 1);
    auto run_lo = [&](int split) { return blocks * split / g.splits; };
    // the cursor of loading: this warp's items (entry, run of hidden columns) one after the other, slot by slot
    int load_item = warp, load_b = 0, load_hi = 0;
    const uint8_t *pa = nullptr, *pb = nullptr;
    auto point = [&]() {
        if (load_item >= items) return;
        const int e = entries[3 * (load_item / g.splits)], split = load_item % g.splits;
        load_b = run_lo(split);
        load_hi = run_lo(split + 1);
        pa = g.w_out + ((size_t)e * g.D + ra) * g.ld_out;
        pb = g.w_out + ((size_t)e * g.D + rb) * g.ld_out;
    };
    auto load = [&](int slot) {
        if (load_item >= items) return;
        const uint32_t dst = ring_at + slot * FEW_SLOT;
        const int at = load_b * 128 + t4 * 16;
        few_copy16(dst, pa, at, bytes);
        few_copy16(dst + 512, pb, at, bytes);
        few_copy16(dst + 1024, pa, at + 64, bytes);
        few_copy16(dst + 1536, pb, at + 64, bytes);
        if (++load_b == load_hi) {
            load_item += FEW_WARPS;
            point();
        }
    };
    point();
#pragma unroll 1
    for (int i = 0; i < FEW_RING; ++i) {
        load(i);
        few_commit();
    }
    if (FP8) {
        const int uf = g.F / 8;
        for (int p0 = warp * 8; p0 < pairs; p0 += FEW_WARPS * 8) {       // four lanes a pair
            const int p = min(p0 + gr, pairs - 1);
            uint32_t big = 0;
#pragma unroll 8
            for (int i = t4; i < uf; i += 4) big = max(big, g.largest[(size_t)p * uf + i]);
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
            if (t4 == 0) largest[p] = big;
        }
        __syncthreads();
    }
    int slot = 0;
    for (int item = warp; item < items; item += FEW_WARPS) {
        const int entry = item / g.splits, split = item % g.splits, e = entries[3 * entry], first = entries[3 * entry + 1], count = entries[3 * entry + 2];
        const float* rows[G];
        float scale[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
            const int pair = places[first + min(j * 8 + gr, count - 1)];
            rows[j] = g.hidden + (size_t)pair * g.F + t4 * (PER / 8);
            scale[j] = FP8 ? f16_scale(largest[pair]) : 1.0f;
        }
        const float* sw = FP8 ? g.s_out + ((size_t)e * db + min(n0, g.D - 1) / 128) * fb : nullptr;
        float acc[G][4];
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
        // the first eight columns' hidden numbers of a block (more columns are rare and read when they are multiplied), a block ahead
        constexpr int HW = FP8 ? 4 : 2;                  // groups of four numbers beside 16 bytes of a weight row
        float4 next[2][HW];
        auto fetch = [&](int j, int b, int h, int i) {
            const int k = b * PER + h * (PER / 2) + i * 4;
            return j * 8 + gr < count && k + t4 * (PER / 8) < g.F ? *reinterpret_cast<const float4*>(rows[j] + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);      // (F is a multiple of 8)
        };
        const int lo = run_lo(split), hi = run_lo(split + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < HW; ++i) next[h][i] = fetch(0, lo, h, i);
        float s_next = FP8 ? sw[lo] : 1.0f;
#pragma unroll 1
        for (int b = lo; b < hi; ++b) {
            // the operand's pairs: fp16, or two bf16 parts
            uint2 high[2][HW], low[2][FP8 ? 1 : HW];
            auto split_up = [&](float4 v, float sc, uint2& p, uint2& r) {
                if (FP8) {
                    p = make_uint2(pair_f16(v.x * sc, v.y * sc), pair_f16(v.z * sc, v.w * sc));
                } else {
                    p = make_uint2(pair_bf16(v.x, v.y), pair_bf16(v.z, v.w));
                    r = make_uint2(pair_bf16(v.x - low_of(p.x), v.y - high_of(p.x)), pair_bf16(v.z - low_of(p.y), v.w - high_of(p.y)));
                }
            };
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < HW; ++i) split_up(next[h][i], scale[0], high[h][i], low[h][FP8 ? 0 : i]);
            const float s0 = s_next;
            if (b + 1 < hi) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < HW; ++i) next[h][i] = fetch(0, b + 1, h, i);
                if (FP8) s_next = sw[b + 1];
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(FEW_RING - 1) : "memory");
            const unsigned char* at = ring + slot * FEW_SLOT + lane * 16;
            float c[G][2][4];
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) c[j][i >> 2][i & 3] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 wl = *reinterpret_cast<const uint4*>(at + 1024 * h), wh = *reinterpret_cast<const uint4*>(at + 512 + 1024 * h);
                const uint32_t lw[4] = {wl.x, wl.y, wl.z, wl.w}, hw[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
                for (int i = 0; i < HW; ++i) {
                    uint32_t a0, a1, a2, a3;
                    if (FP8) {
                        f16_of(lw[i], a0, a2);
                        f16_of(hw[i], a1, a3);
                    } else {
                        a0 = lw[2 * i];
                        a2 = lw[2 * i + 1];
                        a1 = hw[2 * i];
                        a3 = hw[2 * i + 1];
                    }
#pragma unroll
                    for (int j = 0; j < G; ++j) {
                        if (j > 0 && count <= 8 * j) break;
                        uint2 p = high[h][i], r = low[h][FP8 ? 0 : i];
                        if (j > 0) split_up(fetch(j, b, h, i), scale[j], p, r);
                        if (FP8) {
                            mma_f16_f32(c[j][h], a0, a1, a2, a3, p.x, p.y);
                        } else {
                            mma_bf16_f32(acc[j], a0, a1, a2, a3, p.x, p.y);
                            mma_bf16_f32(c[j][1], a0, a1, a2, a3, r.x, r.y);
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] = FP8 ? fmaf(s0, c[j][0][i] + c[j][1][i], acc[j][i]) : acc[j][i] + c[j][1][i];
            load(slot);
            few_commit();
            slot = slot + 1 == FEW_RING ? 0 : slot + 1;
        }
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = j * 8 + t4 * 2 + c;
                if (col >= count) continue;
                const int pair = places[first + col];
                const float back = FP8 ? f16_unscale(largest[pair]) : 1.0f;
                float* at = sums + ((size_t)split * pairs + pair) * 16 + gr;
                at[0] = acc[j][c] * back;
                at[8] = acc[j][2 + c] * back;
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * g.n; i += FEW_THREADS) {
        const int row = i & 15, t = i >> 4;
        if (n0 + row >= g.D) continue;
        float total = 0.0f;
        for (int c = 0; c < g.top; ++c) {
            float y = 0.0f;
            for (int s = 0; s < g.splits; ++s) y += sums[((size_t)s * pairs + t * g.top + c) * 16 + row];
            total = fmaf(wts[t * g.top + c], y, total);
        }
        g.out[(size_t)t * g.D + n0 + row] = __float2bfloat16_rn(total);
    }
}

size_t in_smem(const FewArgs& g) {
    const int tok = g.n <= 8 ? 8 : 16, pairs = g.n * g.top;
    return (size_t)FEW_WARPS * FEW_RING * FEW_SLOT + 4 * ((size_t)2 * FEW_WARPS * 16 * tok + ((g.n * g.E + 3) & ~3) + 6 * pairs + 2 * FEW_WARPS + 2 + FEW_TOKENS);
}
size_t in_x_bytes(const FewArgs& g, bool fp8) { return 4 * (size_t)few_pad(g.n, g.E, g.n * g.top) + 2 * (size_t)g.n * few_x_stride(g.D, fp8); }
size_t out_smem(const FewArgs& g) {
    const int pairs = g.n * g.top;
    return (size_t)FEW_WARPS * FEW_RING * FEW_SLOT + 4 * ((size_t)g.splits * pairs * 16 + 6 * pairs);
}

constexpr size_t FEW_SMEM = 227 * 1024;

template <bool FP8, int G, bool XS>
int launch(FewArgs& g, cudaStream_t s) {
    constexpr size_t most = FEW_SMEM;
    const size_t smem_in = in_smem(g) + (XS ? in_x_bytes(g, FP8) : 0), smem_out = out_smem(g);
    MM_REQUIRE(smem_in <= most && smem_out <= most, "moe few: too many experts or choices for the kernels' shared memory");
    if (!mm_allow_smem<few_in_kernel<FP8, G, XS>>(most) || !mm_allow_smem<few_out_kernel<FP8, G>>(most)) {
        mm_set_last_error("moe few: cannot reserve shared memory");
        return MM_ERR_LAUNCH;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = smem_in;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = FEW_CLUSTER;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // as many clusters as are resident at once, or as there are units for
    static std::atomic<int> resident{0};
    int fit = resident.load(std::memory_order_relaxed);
    if (fit == 0) {
        cfg.gridDim = dim3(FP8_SM_COUNT / FEW_CLUSTER * FEW_CLUSTER);
        if (cudaOccupancyMaxActiveClusters(&fit, few_in_kernel<FP8, G, XS>, &cfg) != cudaSuccess || fit < 1) {
            (void)cudaGetLastError();
            fit = FEW_CLUSTERS;
        }
        if (fit > FEW_CLUSTERS) fit = FEW_CLUSTERS;
        resident.store(fit, std::memory_order_relaxed);
    }
    const int most_experts = g.E < g.n * g.top ? g.E : g.n * g.top;
    const long long groups = ((long long)most_experts * (g.F / 8) * g.KS + FEW_WARPS - 1) / FEW_WARPS, clusters = (groups + FEW_CLUSTER - 1) / FEW_CLUSTER;
    cfg.gridDim = dim3((unsigned)(clusters < fit ? clusters : fit) * FEW_CLUSTER);
    cudaLaunchKernelEx(&cfg, few_in_kernel<FP8, G, XS>, g);
    MM_CHECK_LAUNCH();
    mm_launch_dependent(g_mm_pdl != 0, few_out_kernel<FP8, G>, dim3(ceil_div(g.D, 16)), dim3(FEW_THREADS), smem_out, s, g);
    MM_CHECK_LAUNCH();
    return MM_OK;
}

}  // namespace

// x bf16 [n, ldx]; w_router fp32 [E, D]; experts bf16 (s_in, s_out null): w_in [E, 2 F, D] (gate rows then up rows, or with `interleaved` alternating in
// blocks of 8), w_out [E, D, F]; or e4m3 with scales: w_in [E, 2, F, ld_in], w_out [E, D, ld_out].  ld_in, ld_out: bytes of a row.
// out bf16 [n, D].  scratch: pairs * (4 F + F / 2 + 24) + 32 bytes, pairs = n * top, and with e4m3 experts 36 n D more.
MM_EXPORT int mm_moe_few(const void* x, long long ldx, int n, int D, const void* w_router, int E, int top, int groups, int keep, int scoring, const void* correction,
                         int pair_sum, int renorm, float wscale, const void* w_in, const void* s_in, long long ld_in, const void* w_out, const void* s_out, long long ld_out,
                         int F, int act, float limit, int on_input, int interleaved, void* out, void* scratch, void* stream) {
    MM_REQUIRE(n >= 0 && n <= FEW_TOKENS, "moe few: at most 16 tokens");
    MM_REQUIRE(E > 0 && E <= FEW_MAX_EXPERTS && top > 0 && top <= FEW_MAX_TOP, "moe few: at most 512 experts and 32 choices");
    MM_REQUIRE(groups > 0 && E % groups == 0 && keep > 0 && keep <= groups && top <= keep * (E / groups),
               "moe few: experts must split into equal runs, 0 < keep <= runs, and top fits into the kept runs");
    MM_REQUIRE(scoring == 0 || scoring == 1, "moe few: the scoring is 0 (softmax) or 1 (sigmoid)");
    MM_REQUIRE(act >= 0 && act <= MM_GLU_GELU_TANH, "moe few: unknown activation");
    const bool fp8 = s_in != nullptr;
    MM_REQUIRE(fp8 == (s_out != nullptr) && !(fp8 && interleaved), "moe few: both matrices are in bf16 or both in 8 bits");
    MM_REQUIRE(D > 0 && F > 0 && D % 8 == 0 && F % 8 == 0 && ldx % 8 == 0 && ldx >= 0, "moe few: widths and row strides must be multiples of 8");
    MM_REQUIRE(ld_in % 16 == 0 && ld_out % 16 == 0 && ld_in >= (fp8 ? D : 2 * (long long)D) && ld_out >= (fp8 ? F : 2 * (long long)F), "moe few: weight rows must start on 16-byte boundaries");
    MM_REQUIRE((((uintptr_t)x | (uintptr_t)w_router | (uintptr_t)w_in | (uintptr_t)w_out | (uintptr_t)scratch) & 15) == 0, "moe few: tensors must start on 16-byte boundaries");
    MM_REQUIRE((long long)E * (F / 8) < 0x3fffffff && D < (1 << 28) && F < (1 << 28), "moe few: too large");
    if (n == 0) return MM_OK;
    FewArgs g = {};
    const size_t pairs = (size_t)n * top;
    g.x = (const __nv_bfloat16*)x;
    g.ldx = ldx;
    g.w_router = (const float*)w_router;
    g.correction = (const float*)correction;
    g.w_in = (const uint8_t*)w_in;
    g.w_out = (const uint8_t*)w_out;
    g.s_in = (const float*)s_in;
    g.s_out = (const float*)s_out;
    g.ld_in = ld_in;
    g.ld_out = ld_out;
    g.hidden = (float*)scratch;
    g.largest = (uint32_t*)(g.hidden + pairs * F);
    g.weights = (float*)(g.largest + pairs * (F / 8));
    g.lists = (int32_t*)(g.weights + pairs);
    g.x_half = (uint16_t*)(((uintptr_t)(g.lists + 1 + 4 * pairs) + 15) & ~(uintptr_t)15);
    g.out = (__nv_bfloat16*)out;
    g.n = n;
    g.D = D;
    g.E = E;
    g.top = top;
    g.groups = groups;
    g.keep = keep;
    g.scoring = scoring;
    g.renorm = renorm;
    g.pair_sum = pair_sum;
    g.wscale = wscale;
    g.F = F;
    g.act = act;
    g.limit = limit;
    g.on_input = on_input;
    g.interleaved = interleaved;
    const int in_blocks = (int)(((fp8 ? 1LL : 2LL) * D + 127) / 128), out_blocks = (int)(((fp8 ? 1LL : 2LL) * F + 127) / 128);
    g.KS = 8;
    while (g.KS > in_blocks) g.KS /= 2;
    g.splits = (FEW_WARPS + top - 1) / top;          // a run for every warp when there is one token
    if (g.splits > out_blocks) g.splits = out_blocks;
    cudaStream_t s = (cudaStream_t)stream;
    const bool xs = in_smem(g) + in_x_bytes(g, fp8) <= FEW_SMEM;
    if (fp8) {
        if (xs) return n <= 8 ? launch<true, 1, true>(g, s) : launch<true, 2, true>(g, s);
        return n <= 8 ? launch<true, 1, false>(g, s) : launch<true, 2, false>(g, s);
    }
    if (xs) return n <= 8 ? launch<false, 1, true>(g, s) : launch<false, 2, true>(g, s);
    return n <= 8 ? launch<false, 1, false>(g, s) : launch<false, 2, false>(g, s);
}
