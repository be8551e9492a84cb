// A whole routed-experts layer for up to 16 tokens in two launches.
//
//   z = x W_router^T;  the choice of `top` experts and their weights (moe_route.cuh)
//   h[t, c] = act(W_gate[e] x_t, W_up[e] x_t),   out[t] = sum over the choices c in order of wts[t, c] W_down[e] h[t, c],   e = idx[t, c].
//
// A few tokens are bound by the chosen experts' matrices: each is read once, by mma.sync with 16 weight rows as the 16-row operand and the expert's
// rows of x, found by their places, as its 8 (or twice 8) columns.  Nothing is sorted or copied.
//
// First launch, clusters of eight CTAs: every cluster makes all logits (an eighth of the router's rows each) and the choice (every eighth token each), handed
// round over distributed shared memory; every CTA makes the list of experts with their tokens, then its share of the units of 8 gate and 8 up rows.
// That costs a read of the router per cluster from L2 and saves a launch and its wait for another.
// Second launch: 16 output columns a CTA; its warps share out the experts' runs of hidden columns, whose sums are kept apart per (token, choice) and added
// in the order of the choice.  A token's output does not depend on the others: every sum is cut by the layer's sizes alone.
//
// The router's weights are fp32: each is three bf16 parts (hi, mid, lo, 24 bits together), x is bf16, the sums are fp32.
// Experts in bf16: x as it is, the fp32 hidden rows as two bf16 parts (2^-17 of a number is lost).
// Experts in e4m3 with a scale per block of 128 x 128: a row of x, after a power of two that brings its largest number to 2^7 .. 2^8, is two e4m3 parts, hi and
// 16 lo: together bf16's eight bits (a number below 2^-13 of the row's largest loses what is below 2^-21 of it).  Four tokens' parts are the eight
// columns, so the weights are multiplied as they lie.  The hidden rows become two fp16 parts (22 bits) after a power of two that brings their largest number
// to 2^14 .. 2^15, beside the weights in fp16, exactly.  (One part, 11 bits, moved one result in ten to the neighbouring bf16 number; the second takes 1 token
// from 25.8 to 26.0 us, 8 tokens from 71.4 to 74.8, 16 tokens from 97.7 to 103.5.)
//
// Bound by memory for the experts' matrices (one token, 128 experts of 768 and 2,048 wide, 8 of them, in 8 bits: 38 MB, 5.9 us), but the fixed parts weigh as much:
// the router about 5 us (830 cycles a step and warp, of loads in a ring or not, of conversions or not), the choice 3, cluster barriers and set-up 3, the second
// launch's set-up 3; then 700 to 1,000 cycles a warp for 2 KB, the latency of a block's own instructions (a ring of six slots takes the same, half a depth a warp
// no less).  As captured, one input again and again: 1 token 26 us (27.5 with other inputs in turn), 8 tokens 72 to 79, 16 tokens 103 to 112 on 76 to 83 experts (floor 59.6); 8 tokens
// on 16 experts of 1,408 in bf16, 4 each, 60 (38.1).
#include <cuda_fp16.h>

#include "fp8.cuh"
#include "fp8_launch.h"
#include "moe_route.cuh"

namespace {

constexpr int FEW_THREADS = 512, FEW_WARPS = 16, FEW_RING = 3, FEW_SLOT = 2048, FEW_CLUSTER = 8;
constexpr int FEW_TOKENS = 16, FEW_MAX_EXPERTS = 512, FEW_MAX_TOP = 32;
constexpr int FEW_RANK_EXPERTS = 192;    // up to here a token's scores are ranked all at once, beyond by searches
constexpr int FEW_ROWS = 8;              // (token, choice) rows of an entry; an expert with more has several
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
    uint8_t* x_copy;                      // [clusters][n][few_x_bytes]: x as the products read it, where it does not fit into shared memory
    __nv_bfloat16* out;
    long long ldx, ld_in, ld_out;
    int n, D, E, top, groups, keep, scoring, renorm, pair_sum, F, act, on_input, interleaved;
    float wscale, limit;
    int KS, splits;
};

__device__ __forceinline__ void few_copy16(uint32_t dst, const uint8_t* src, int left) {      // the first `left` of 16 bytes, noughts behind them
    const int n = min(max(left, 0), 16);
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(n > 0 ? src : src - (16 - left + 15) / 16 * 16), "r"(n) : "memory");
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
// how far a pair of fp16 numbers is above (x, y), as a pair
__device__ __forceinline__ uint32_t f16_excess(uint32_t pair, float x, float y) {
    float a, b;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.f16 %0, l, %3;\n\tsub.rn.f32.f16 %1, h, %4;\n\t}" : "=f"(a), "=f"(b) : "r"(pair), "f"(x), "f"(y));
    return pair_f16(a, b);
}
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }
__device__ __forceinline__ float low_of(uint32_t bf16_pair) { return __uint_as_float(bf16_pair << 16); }
__device__ __forceinline__ float high_of(uint32_t bf16_pair) { return __uint_as_float(bf16_pair & 0xffff0000u); }
__device__ __forceinline__ float2 times(float x, float y, float s) {       // two products in one instruction
    uint64_t v = ((uint64_t)__float_as_uint(y) << 32) | __float_as_uint(x);
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(v) : "l"(((uint64_t)__float_as_uint(s) << 32) | __float_as_uint(s)));
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ void mma_e4m3_f32(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four e4m3 numbers as two fp16 pairs
__device__ __forceinline__ void f16_of(uint32_t w, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(a), "=r"(b) : "r"(w));
}

// a word into the same place of a CTA of the cluster
__device__ __forceinline__ void st_cluster(void* at, uint32_t cta, uint32_t v) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(cta));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(v) : "memory");
}
__device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The power of two that brings a size to 2^to .. 2^(to + 1) (sizes next to the smallest normal number: as far as it goes), and its inverse; an infinity or
// a NaN stays one under it.
__device__ __forceinline__ int few_exponent(uint32_t size_bits) { return min(max((int)(size_bits >> 23), 16), 254); }
__device__ __forceinline__ float few_scale(uint32_t size_bits, int to) { return __uint_as_float((uint32_t)(254 + to - few_exponent(size_bits)) << 23); }
__device__ __forceinline__ float few_unscale(uint32_t size_bits, int to) { return __uint_as_float((uint32_t)(few_exponent(size_bits) - to) << 23); }
constexpr int X_TO = 7, HIDDEN_TO = 14;

static_assert(4 * (4 * (FEW_MAX_EXPERTS + FEW_MAX_TOP) + FEW_MAX_EXPERTS) <= FEW_WARPS * FEW_RING * FEW_SLOT && 2 * 8 * 2 * FEW_MAX_EXPERTS <= FEW_WARPS * FEW_RING * FEW_SLOT,
              "the choice's scratch and the experts' first places stand where the rings start later");

// moe_route_warp's scores (the same formula), and their order as numbers: 0 is not to be chosen (a NaN, minus infinity).  A warp; s, key: E words each.
// (Code that runs once in a launch is fetched from L2 as it goes: short loops beat unrolled ones here.)
__device__ __forceinline__ void few_scores(const float* __restrict__ z, float* s, uint32_t* key, int lane, int E, int scoring, const float* __restrict__ correction) {
    float m = 0.0f, inv = 1.0f;
    if (scoring == 0) {
        m = -INFINITY;
#pragma unroll 2
        for (int e = lane; e < E; e += 32) m = fmaxf(m, z[e]);
        m = warp_max(m);
        float sum = 0.0f;
#pragma unroll 2
        for (int e = lane; e < E; e += 32) {
            const float p = expf(z[e] - m);
            s[e] = p;
            sum += p;
        }
        inv = 1.0f / warp_sum(sum);
    }
#pragma unroll 2
    for (int e = lane; e < E; e += 32) {
        const float v = scoring == 1 ? 1.0f / (1.0f + expf(-z[e])) : s[e] * inv;
        s[e] = v;
        const float c = correction ? v + correction[e] : v;
        const uint32_t u = __float_as_uint(c);
        key[e] = c != c || c == -INFINITY ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
    }
    for (int e = E + lane; e < (E + 3) / 4 * 4; e += 32) key[e] = 0;
}

// A warp: the choice by `top` searches for the largest number, the lowest expert among equals; chosen[k] = expert, or -1 where fewer can be chosen.
__device__ __forceinline__ void few_search(uint32_t* key, int lane, int E, int top, int32_t* chosen) {
#pragma unroll 1
    for (int k = 0; k < top; ++k) {
        uint32_t best = 0;
        int at = 0x7fffffff;
#pragma unroll 4
        for (int e = lane; e < E; e += 32) {
            const uint32_t v = key[e];
            if (v > best) {
                best = v;
                at = e;
            }
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        const int e = (int)__reduce_min_sync(0xffffffffu, best == most && most != 0 ? (uint32_t)at : 0x7fffffffu);
        if (lane == 0) chosen[k] = e == 0x7fffffff ? -1 : e;
        if (e != 0x7fffffff && (e & 31) == lane) key[e] = 0;
        __syncwarp();
    }
}

// A slot of a warp's ring: 128 bytes of 16 weight rows (a lane's four pieces: bytes t * 16 .. + 15 and 64 on of rows g and g + 8), 128 e4m3 or 64
// bf16 numbers a row.  The order of k inside it is free as long as both operands agree: a lane's pieces are multiplied as they lie.

// Bytes of a row of x as the products read it, noughts behind its end, rows of neighbouring columns in different banks.  e4m3: hi numbers, then lo.
__host__ __device__ inline int few_part_bytes(int D) { return (D + 127) / 128 * 128 + 32; }
__host__ __device__ inline int few_x_bytes(int D, bool fp8) { return fp8 ? 2 * few_part_bytes(D) : (D + 63) / 64 * 128 + 64; }
// 4-byte words of the first launch's lists, whole 16 bytes
__host__ __device__ inline int few_list_words(int n, int E, int pairs) { return (((n * E + 3) & ~3) + 6 * pairs + 2 * FEW_WARPS + 2 + FEW_TOKENS + 3) & ~3; }

// ---------------------------------------------------------------------------------------------------------------
// first launch: router, choice, gate and up products, activation
// ---------------------------------------------------------------------------------------------------------------
template <bool FP8, bool XS>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_in_kernel(const __grid_constant__ FewArgs g) {
    constexpr int NG = FP8 ? 2 : 1, COLS = 8 * NG;                                              // columns of a unit: groups of eight
    extern __shared__ __align__(16) unsigned char few_smem[];
    unsigned char* rings = few_smem;                                                            // until they start: the choice's scratch
    float* part = reinterpret_cast<float*>(few_smem + FEW_WARPS * FEW_RING * FEW_SLOT);         // [2][16 warps][16][COLS]; the router's: [16 warps][16][16]
    float* logits = part + (FP8 ? 2 : 1) * FEW_WARPS * 16 * 16;                                 // [n][E]
    const int pairs = g.n * g.top;
    int32_t* idx = reinterpret_cast<int32_t*>(logits + ((g.n * g.E + 3) & ~3));                 // [pairs]
    float* wts = reinterpret_cast<float*>(idx + pairs);                                         // [pairs]
    int32_t* places = reinterpret_cast<int32_t*>(wts + pairs);                                  // [pairs]: the pair at every place, by expert
    int32_t* entries = places + pairs;                                                          // [pairs][3]
    int32_t* sums = entries + 3 * pairs;                                                        // [2][16 warps], [2] totals
    uint32_t* x_largest = reinterpret_cast<uint32_t*>(sums + 2 * FEW_WARPS + 2);                // [16]
    const int x_bytes = few_x_bytes(g.D, FP8);
    uint8_t* x_rows = XS ? reinterpret_cast<uint8_t*>(logits + few_list_words(g.n, g.E, pairs)) : g.x_copy + (size_t)(blockIdx.x / FEW_CLUSTER) * g.n * x_bytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t4 = lane & 3;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    pdl_trigger();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // waited for in front of the first store to another CTA: by then it runs

    if (FP8 && threadIdx.x < FEW_TOKENS) x_largest[threadIdx.x] = 0;
    // ---- logits: 16 experts a tile, a sixteenth of the depth a warp; and the rows' largest sizes ----
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    __syncthreads();
    {
        constexpr int BATCH = 4, STEP_BYTES = 32 * 48;          // steps of 16 that are on their way together: what a lane multiplies of them, in its own places
        static_assert(BATCH * STEP_BYTES <= FEW_RING * FEW_SLOT, "a warp's share of the rings");
        const int steps = (g.D + 15) / 16, lo = steps * warp / FEW_WARPS, hi = steps * (warp + 1) / FEW_WARPS;
        unsigned char* mine_at = rings + warp * FEW_RING * FEW_SLOT + lane * 16;
        const uint32_t stage = (uint32_t)__cvta_generic_to_shared(mine_at);
        const __nv_bfloat16 *xa = g.x + (size_t)min(gr, g.n - 1) * g.ldx, *xb = g.x + (size_t)min(gr + 8, g.n - 1) * g.ldx;      // (columns without a token: not looked at)
        uint32_t big0 = 0, big1 = 0;
#pragma unroll 1
        for (int tile = rank; tile * 16 < g.E || (FP8 && tile == (int)rank); tile += FEW_CLUSTER) {      // (a CTA without a tile still looks at x)
            const float *wa = g.w_router + (size_t)min(tile * 16 + gr, g.E - 1) * g.D, *wb = g.w_router + (size_t)min(tile * 16 + gr + 8, g.E - 1) * g.D;
            float acc[2][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[0][c] = acc[1][c] = 0.0f;
auto load = [&](int s, int i) {
                const int k = s * 16 + t4 * 4, on = s < hi && k < g.D ? 1 : 0;       // (D is a multiple of 8)
                const uint32_t dst = stage + i * STEP_BYTES;
                const float *pa = wa + (on ? k : 0), *pb = wb + (on ? k : 0);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(pa), "r"(on * 16) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 512), "l"(pb), "r"(on * 16) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + 1024), "l"(xa + (on ? k : 0)), "r"(on * 8) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + 1032), "l"(xb + (on ? k : 0)), "r"(on * 8) : "memory");
                few_commit();
            };
#pragma unroll 1
            for (int i = 0; i < BATCH; ++i) load(lo + i, i);
#pragma unroll 1
            for (int s = lo, i = 0; s < hi; ++s, i = i + 1 == BATCH ? 0 : i + 1) {
                asm volatile("cp.async.wait_group %0;" ::"n"(BATCH - 1) : "memory");
                const unsigned char* at = mine_at + i * STEP_BYTES;
                const float4 a = *reinterpret_cast<const float4*>(at), b = *reinterpret_cast<const float4*>(at + 512);
                const uint4 xv = *reinterpret_cast<const uint4*>(at + 1024);
                load(s + BATCH, i);
                float r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int p = 0; p < 3; ++p) {       // hi, mid, lo: eight bits each, cut off, so that nothing is lost
                    const uint32_t a0 = upper_halves(r[0], r[1]), a2 = upper_halves(r[2], r[3]), a1 = upper_halves(r[4], r[5]), a3 = upper_halves(r[6], r[7]);
                    if (p < 2) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) r[c] -= high_of(__float_as_uint(r[c]));      // exact
                    }
                    mma_bf16_f32(acc[0], a0, a1, a2, a3, xv.x, xv.y);
                    if (g.n > 8) mma_bf16_f32(acc[1], a0, a1, a2, a3, xv.z, xv.w);
                }
                if (FP8) {
                    big0 = max(big0, max(max((xv.x & 0x7fffu) << 16, xv.x & 0x7fff0000u), max((xv.y & 0x7fffu) << 16, xv.y & 0x7fff0000u)));
                    big1 = max(big1, max(max((xv.z & 0x7fffu) << 16, xv.z & 0x7fff0000u), max((xv.w & 0x7fffu) << 16, xv.w & 0x7fff0000u)));
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");       // (nothing lands behind this: the bytes are used for other things)
            float* mine = part + (warp * 16 + gr) * 16 + t4 * 2;
            __syncthreads();        // the tile before has been read
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                *reinterpret_cast<float2*>(mine + j * 8) = make_float2(acc[j][0], acc[j][1]);
                *reinterpret_cast<float2*>(mine + 128 + j * 8) = make_float2(acc[j][2], acc[j][3]);
            }
            __syncthreads();
            if (threadIdx.x < 16 * g.n) {
                const int row = threadIdx.x & 15, tok = threadIdx.x >> 4, e = tile * 16 + row;
                float z = 0.0f;
#pragma unroll
                for (int w = 0; w < FEW_WARPS; ++w) z += part[(w * 16 + row) * 16 + tok];
                if (e < g.E) st_cluster(logits + tok * g.E + e, tok % FEW_CLUSTER, __float_as_uint(z));      // to the CTA that chooses for the token
            }
        }
        if (FP8) {
            if (gr < g.n) atomicMax(x_largest + gr, big0);
            if (gr + 8 < g.n) atomicMax(x_largest + gr + 8, big1);
        }
    }
    // ---- x as the products read it: into shared memory, or (rows too long for that) the cluster's own copy in memory, an eighth by every CTA ----
    __syncthreads();        // (x_largest; the rings' bytes)
    {
        const int chunks = FP8 ? few_part_bytes(g.D) / 8 - 4 : (g.D + 63) / 64 * 8, step = XS ? FEW_THREADS : FEW_CLUSTER * FEW_THREADS;
#pragma unroll 2
        for (int i = XS ? threadIdx.x : rank * FEW_THREADS + threadIdx.x; i < g.n * chunks; i += step) {
            const int t = i / chunks, d = (i - t * chunks) * 8;
            const uint4 v = d < g.D ? *reinterpret_cast<const uint4*>(g.x + (size_t)t * g.ldx + d) : make_uint4(0, 0, 0, 0);
            uint8_t* row = x_rows + (size_t)t * x_bytes;
            if (FP8) {
                const float s = few_scale(x_largest[t], X_TO);
                const bool number = x_largest[t] < 0x7f800000u;      // else the row is NaN: a conversion would make a number of an infinity
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                uint32_t hi[2] = {0x7f7f7f7fu, 0x7f7f7f7fu}, lo[2] = {0x7f7f7f7fu, 0x7f7f7f7fu};
                if (number) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float f[4] = {low_of(w[2 * j]) * s, high_of(w[2 * j]) * s, low_of(w[2 * j + 1]) * s, high_of(w[2 * j + 1]) * s};
                        hi[j] = fp8_pack4(f[0], f[1], f[2], f[3]);
                        uint32_t p, q;
                        f16_of(hi[j], p, q);
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&p)), b = __half22float2(*reinterpret_cast<const __half2*>(&q));
                        lo[j] = fp8_pack4((f[0] - a.x) * 16.0f, (f[1] - a.y) * 16.0f, (f[2] - b.x) * 16.0f, (f[3] - b.y) * 16.0f);
                    }
                }
                *reinterpret_cast<uint2*>(row + d) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(row + few_part_bytes(g.D) + d) = make_uint2(lo[0], lo[1]);
            } else {
                *reinterpret_cast<uint4*>(row + 2 * d) = v;
            }
        }
    }
    cluster_barrier();
    // ---- the choice, every eighth token here, for the whole cluster ----
    const int own_tokens = ((int)g.n - (int)rank + FEW_CLUSTER - 1) / FEW_CLUSTER;             // tokens rank, rank + 8
    if (g.keep == g.groups) {
        const int Ew = (g.E + 3) & ~3;
        float* scores = reinterpret_cast<float*>(rings);                                        // [2][Ew]
        uint32_t* keys = reinterpret_cast<uint32_t*>(scores + 2 * Ew);                          // [2][Ew]
        int32_t* chosen = reinterpret_cast<int32_t*>(keys + 2 * Ew);                            // [2][top]
        if (warp < own_tokens) few_scores(logits + (rank + warp * FEW_CLUSTER) * g.E, scores + warp * Ew, keys + warp * Ew, lane, g.E, g.scoring, g.correction);
        if (threadIdx.x < own_tokens * g.top) chosen[threadIdx.x] = -1;
        __syncthreads();
        if (g.E <= FEW_RANK_EXPERTS) {
            // four threads per token and expert count the scores ahead of its own (equal ones of lower experts are); own_tokens * Ew is a multiple of 4, and
            // a warp's eight are in the loop together up to the last: the others count for the last one
#pragma unroll 1
            for (int i0 = warp * 8; i0 < own_tokens * Ew; i0 += FEW_WARPS * 8) {
                const int i = min(i0 + (lane >> 2), own_tokens * Ew - 1), t = i / Ew, e = i - t * Ew;
                const uint32_t* key = keys + t * Ew;
                const uint32_t own = key[e];
                int ahead = 0;
#pragma unroll 2
                for (int o = (lane & 3) * 4; o < Ew; o += 16) {
                    const uint4 v = *reinterpret_cast<const uint4*>(key + o);
                    const uint32_t least = own - (o < e ? 1u : 0u);      // (own > 0 where it counts; the four beside e itself: below)
                    ahead += (v.x > least) + (v.y > least) + (v.z > least) + (v.w > least);
                }
                ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
                ahead += __shfl_xor_sync(0xffffffffu, ahead, 2);
                // the group of four around e was compared as if all of it stood before e: itself, and equals behind it, are taken back
                if (own != 0 && (lane & 3) == 0) {
                    if ((e & 3) != 0)
                        for (int o = e; o < (e | 3) + 1; ++o) ahead -= key[o] == own;
                    if (ahead < g.top) chosen[t * g.top + ahead] = e;
                }
            }
        } else if (warp < own_tokens) {
            few_search(keys + warp * Ew, lane, g.E, g.top, chosen + warp * g.top);
        }
        __syncthreads();
        if (warp < own_tokens) {
            // the weights, summed in the order of the choice; fewer to choose from than `top`: the rest is expert 0 without a weight
            const int e = lane < g.top ? chosen[warp * g.top + lane] : -1;
            const float w = e >= 0 ? scores[warp * Ew + e] : 0.0f;
            float total = 0.0f;
#pragma unroll 2
            for (int k = 0; k < g.top; ++k) total += __shfl_sync(0xffffffffu, w, k);
            if (lane < g.top) {
                const int at = (rank + warp * FEW_CLUSTER) * g.top + lane;
                const float weight = g.renorm || g.wscale != 1.0f ? w / (g.renorm ? total + 1e-20f : 1.0f) * g.wscale : w;
#pragma unroll 1
                for (int c = 0; c < FEW_CLUSTER; ++c) {
                    st_cluster(idx + at, c, (uint32_t)max(e, 0));
                    st_cluster(wts + at, c, __float_as_uint(weight));
                }
            }
        }
    } else if (warp < own_tokens) {
        const int t = rank + warp * FEW_CLUSTER;
        int32_t* chosen = places + t * g.top;                   // (not in use yet)
        float* weight = reinterpret_cast<float*>(entries) + t * g.top;
        moe_route_warp(logits + t * g.E, reinterpret_cast<float*>(rings) + (size_t)warp * 2 * (g.E + g.groups), lane, g.E, g.top, g.groups, g.keep, places,
                       reinterpret_cast<float*>(entries), (size_t)t, g.scoring, g.correction, g.pair_sum, g.renorm, g.wscale);
        __syncwarp();
        if (lane < g.top)
            for (int c = 0; c < FEW_CLUSTER; ++c) {
                st_cluster(idx + t * g.top + lane, c, (uint32_t)chosen[lane]);
                st_cluster(wts + t * g.top + lane, c, __float_as_uint(weight[lane]));
            }
    }
    cluster_barrier();       // (nobody reaches into another CTA behind this)
    // ---- the experts that someone chose, in order, with their pairs (token * top + choice): a thread per expert counts, a thread per pair finds its place ----
    {
        const int e = threadIdx.x, mine = threadIdx.x < pairs ? idx[threadIdx.x] : -1;
        int count = 0, before = 0;
#pragma unroll 2
        for (int p = 0; p + 4 <= pairs; p += 4) {
            const int4 v = *reinterpret_cast<const int4*>(idx + p);
            count += (v.x == e) + (v.y == e) + (v.z == e) + (v.w == e);
            before += (v.x == mine && p < e) + (v.y == mine && p + 1 < e) + (v.z == mine && p + 2 < e) + (v.w == mine && p + 3 < e);
        }
        for (int p = pairs & ~3; p < pairs; ++p) {
            const int v = idx[p];
            count += v == e;
            before += v == mine && p < e;
        }
        if (e >= g.E) count = 0;
        const int parts = (count + FEW_ROWS - 1) / FEW_ROWS;
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
#pragma unroll 4
        for (int w = 0; w < warp; ++w) {
            first += sums[w];
            entry += sums[FEW_WARPS + w];
        }
        if (threadIdx.x == FEW_THREADS - 1) sums[2 * FEW_WARPS] = entry + parts;
        int32_t* firsts = reinterpret_cast<int32_t*>(rings) + 4 * (FEW_MAX_EXPERTS + FEW_MAX_TOP);      // [E], behind the scores
        if (e < g.E) firsts[e] = first;
        for (int i = 0; i < parts; ++i) {
            entries[3 * (entry + i)] = e;
            entries[3 * (entry + i) + 1] = first + i * FEW_ROWS;
            entries[3 * (entry + i) + 2] = min(FEW_ROWS, count - i * FEW_ROWS);
        }
        __syncthreads();
        if (mine >= 0) places[firsts[mine] + before] = threadIdx.x;
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
    // warps costs about three)  ----
    const int bytes = FP8 ? g.D : 2 * g.D, blocks = (bytes + 127) / 128, uf = g.F / 8, units = n_entries * uf;
    const int side = FEW_WARPS / g.KS, grid = (int)gridDim.x;
    const bool alone = g.KS == 1 || (units + grid * FEW_WARPS - 1) / (grid * FEW_WARPS) * blocks <= (units + grid * side - 1) / (grid * side) * (blocks / g.KS + 3);
    const int RT = alone ? FEW_WARPS : side, rt = alone ? warp : warp / g.KS, run_lo = alone ? 0 : warp % g.KS, run_hi = alone ? g.KS : run_lo + 1;
    const int lo = blocks * run_lo / g.KS, hi = blocks * run_hi / g.KS, nb = hi - lo;
    // (warps that are alone take every grid's-width unit, so that few units are spread over all CTAs)
    const int stride = grid * RT, unit0 = alone ? (int)blockIdx.x + rt * grid : (int)blockIdx.x * RT + rt;
    const int begin = alone ? unit0 : (int)blockIdx.x * RT, my_steps = begin < units ? (units - 1 - begin) / stride + 1 : 0;
    unsigned char* ring = rings + warp * FEW_RING * FEW_SLOT;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const int kb = (g.D + 127) / 128, fb = (g.F + 127) / 128;
    // a place in the units: (entry, unit of 8 columns), carried along; behind the last unit it stays on it (not stored)
    struct Cursor {
        int entry, fu;
    };
    auto cursor_at = [&](int u) {
        u = min(u, units - 1);
        const int e = u / uf;
        return Cursor{e, u - e * uf};
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
        size_t ra = (size_t)2 * e * g.F + f, rb = ra + g.F;
        if (!FP8 && g.interleaved) {
            ra += f - gr;
            rb = ra + 8;
        }
        pa = g.w_in + ra * g.ld_in + lo * 128 + t4 * 16;
        pb = g.w_in + rb * g.ld_in + lo * 128 + t4 * 16;
    };
    const int total = nb * my_steps;
    const bool whole = bytes % 128 == 0;
    auto load = [&](int slot) {
        const uint32_t dst = ring_at + slot * FEW_SLOT;
        if (whole) {
            few_copy16(dst, pa);
            few_copy16(dst + 512, pb);
            few_copy16(dst + 1024, pa + 64);
            few_copy16(dst + 1536, pb + 64);
        } else {
            const int left = bytes - load_b * 128 - t4 * 16;
            few_copy16(dst, pa, left);
            few_copy16(dst + 512, pb, left);
            few_copy16(dst + 1024, pa + 64, left - 64);
            few_copy16(dst + 1536, pb + 64, left - 64);
        }
        pa += 128;
        pb += 128;
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
        // e4m3: column c of group j is hi of row 4 j + c, column 4 + c its lo.  (Columns without a row: another's numbers, not stored.)
        const uint8_t* rows[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int t = places[first + min(FP8 ? j * 4 + (gr & 3) : gr, count - 1)] / g.top;
            rows[j] = x_rows + (size_t)t * x_bytes + (FP8 && gr >= 4 ? few_part_bytes(g.D) : 0) + t4 * 16 + lo * 128;
        }
        const float *sg = nullptr, *su = nullptr;
        float s0_next = 1.0f, s1_next = 1.0f;
        if (FP8) {
            sg = g.s_in + ((size_t)2 * entries[3 * here.entry] * fb + f0 / 128) * kb;
            su = sg + (size_t)fb * kb;
            s0_next = sg[lo];
            s1_next = su[lo];
        }
        float sum[NG][4];
#pragma unroll
        for (int j = 0; j < NG; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[j][c] = 0.0f;
        int b = lo;
#pragma unroll 1
        for (int run = run_lo; run < run_hi; ++run) {
            float acc[NG][4];
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
            const int end = blocks * (run + 1) / g.KS;
#pragma unroll 1
            for (; b < end; ++b) {
                const float s0 = s0_next, s1 = s1_next;
                if (FP8 && b + 1 < hi) {
                    s0_next = sg[b + 1];
                    s1_next = su[b + 1];
                }
                asm volatile("cp.async.wait_group %0;" ::"n"(FEW_RING - 1) : "memory");
                const unsigned char* at = ring + slot * FEW_SLOT + lane * 16;
                const uint4 l0 = *reinterpret_cast<const uint4*>(at), h0 = *reinterpret_cast<const uint4*>(at + 512);
                const uint4 l1 = *reinterpret_cast<const uint4*>(at + 1024), h1 = *reinterpret_cast<const uint4*>(at + 1536);
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    if (j > 0 && count <= 4) break;
                    const uint4 x0 = *reinterpret_cast<const uint4*>(rows[j]), x1 = *reinterpret_cast<const uint4*>(rows[j] + 64);
                    float c0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, c1[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // two chains: a product's results are 26 cycles away
                    if (FP8) {
                        mma_e4m3_f32(c0, l0.x, h0.x, l0.y, h0.y, x0.x, x0.y);
                        mma_e4m3_f32(c1, l1.x, h1.x, l1.y, h1.y, x1.x, x1.y);
                        mma_e4m3_f32(c0, l0.z, h0.z, l0.w, h0.w, x0.z, x0.w);
                        mma_e4m3_f32(c1, l1.z, h1.z, l1.w, h1.w, x1.z, x1.w);
                    } else {
                        mma_bf16_f32(c0, l0.x, h0.x, l0.y, h0.y, x0.x, x0.y);
                        mma_bf16_f32(c1, l1.x, h1.x, l1.y, h1.y, x1.x, x1.y);
                        mma_bf16_f32(c0, l0.z, h0.z, l0.w, h0.w, x0.z, x0.w);
                        mma_bf16_f32(c1, l1.z, h1.z, l1.w, h1.w, x1.z, x1.w);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[j][i] = FP8 ? fmaf(i < 2 ? s0 : s1, c0[i] + c1[i], acc[j][i]) : acc[j][i] + (c0[i] + c1[i]);
                }
#pragma unroll
                for (int j = 0; j < NG; ++j) rows[j] += 128;
                if (done + FEW_RING < total) load(slot);
                few_commit();
                ++done;
                slot = slot + 1 == FEW_RING ? 0 : slot + 1;
            }
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[j][c] += acc[j][c];
        }
        if (alone) {
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                if (j > 0 && count <= 4) break;
                if (FP8) {       // hi + lo
#pragma unroll
                    for (int c = 0; c < 4; ++c) sum[j][c] = fmaf(__shfl_xor_sync(0xffffffffu, sum[j][c], 2), 0.0625f, sum[j][c]);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = (FP8 ? j * 4 : 0) + t4 * 2 + c;
                    const bool on = col < count && (!FP8 || t4 < 2);
                    const int pair = on ? places[first + col] : 0;
                    float y = sum[j][c], v = sum[j][2 + c];
                    if (FP8) {
                        const float back = few_unscale(x_largest[pair / g.top], X_TO);
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
            float* mine = part + (((step & 1) * FEW_WARPS + warp) * 16 + gr) * COLS + t4 * 2;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                *reinterpret_cast<float2*>(mine + j * 8) = make_float2(sum[j][0], sum[j][1]);
                *reinterpret_cast<float2*>(mine + 8 * COLS + j * 8) = make_float2(sum[j][2], sum[j][3]);
            }
            __syncthreads();
            // eight columns of a pair by eight neighbouring threads; other warps every time
            const float* all = part + (step & 1) * FEW_WARPS * 16 * COLS;
#pragma unroll 1
            for (int i = (threadIdx.x + step * 128) & (FEW_THREADS - 1); i < RT * FEW_ROWS * 8; i += FEW_THREADS) {      // (a multiple of 32)
                const int f = i & 7, j = (i >> 3) % FEW_ROWS, tile = (i >> 3) / FEW_ROWS, unit = (int)blockIdx.x * RT + step * stride + tile;
                const Cursor at = cursor_at(unit);
                const bool on = unit < units && j < entries[3 * at.entry + 2];
                float h = 0.0f;
                int pair = 0;
                if (on) {
                    pair = places[entries[3 * at.entry + 1] + j];
                    const float* p = all + (tile * g.KS * 16 + f) * COLS + (FP8 ? (j >> 2) * 8 + (j & 3) : j);
                    float y = 0.0f, v = 0.0f, yl = 0.0f, vl = 0.0f;
                    for (int s = 0; s < g.KS; ++s) {
                        y += p[s * 16 * COLS];
                        v += p[s * 16 * COLS + 8 * COLS];
                        if (FP8) {
                            yl += p[s * 16 * COLS + 4];
                            vl += p[s * 16 * COLS + 8 * COLS + 4];
                        }
                    }
                    if (FP8) {
                        const float back = few_unscale(x_largest[pair / g.top], X_TO);
                        y = fmaf(yl, 0.0625f, y) * back;
                        v = fmaf(vl, 0.0625f, v) * back;
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
template <bool FP8>
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
    constexpr int PER = FP8 ? 128 : 64, HW = FP8 ? 4 : 2;      // numbers in a slot's row; groups of four numbers beside 16 bytes of a weight row
    const int bytes = FP8 ? g.F : 2 * g.F, blocks = (bytes + 127) / 128, items = n_entries * g.splits, n0 = blockIdx.x * 16;
    const int fb = (g.F + 127) / 128, db = (g.D + 127) / 128;
    const bool whole = bytes % 128 == 0;
    unsigned char* ring = few_smem + warp * FEW_RING * FEW_SLOT;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
    const int ra = min(n0 + gr, g.D - 1), rb = min(n0 + gr + 8, g.D - 1);
    // the cursor of loading: this warp's items (entry, run of hidden columns) one after the other, slot by slot
    int load_item = warp, load_b = 0, load_hi = 0;
    const uint8_t *pa = nullptr, *pb = nullptr;
    auto point = [&]() {
        if (load_item >= items) return;
        const int entry = load_item / g.splits, split = load_item - entry * g.splits, e = entries[3 * entry];
        load_b = blocks * split / g.splits;
        load_hi = blocks * (split + 1) / g.splits;
        pa = g.w_out + ((size_t)e * g.D + ra) * g.ld_out + load_b * 128 + t4 * 16;
        pb = g.w_out + ((size_t)e * g.D + rb) * g.ld_out + load_b * 128 + t4 * 16;
    };
    auto load = [&](int slot) {
        if (load_item >= items) return;
        const uint32_t dst = ring_at + slot * FEW_SLOT;
        if (whole) {
            few_copy16(dst, pa);
            few_copy16(dst + 512, pb);
            few_copy16(dst + 1024, pa + 64);
            few_copy16(dst + 1536, pb + 64);
        } else {
            const int left = bytes - load_b * 128 - t4 * 16;
            few_copy16(dst, pa, left);
            few_copy16(dst + 512, pb, left);
            few_copy16(dst + 1024, pa + 64, left - 64);
            few_copy16(dst + 1536, pb + 64, left - 64);
        }
        pa += 128;
        pb += 128;
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
        if (pairs <= 2 * FEW_WARPS) {
            for (int p = warp; p < pairs; p += FEW_WARPS) {
                uint32_t big = 0;
#pragma unroll 4
                for (int i = lane; i < uf; i += 32) big = max(big, g.largest[(size_t)p * uf + i]);
                big = __reduce_max_sync(0xffffffffu, big);
                if (lane == 0) largest[p] = big;
            }
        } else {
            for (int p0 = warp * 8; p0 < pairs; p0 += FEW_WARPS * 8) {       // four lanes a pair
                const int p = min(p0 + gr, pairs - 1);
                uint32_t big = 0;
#pragma unroll 8
                for (int i = t4; i < uf; i += 4) big = max(big, g.largest[(size_t)p * uf + i]);
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                if (t4 == 0) largest[p] = big;
            }
        }
        __syncthreads();
    }
    // an item under way; the hidden numbers of its next block, or of the next item's first, are fetched a block ahead
    struct Item {
        const float* row;        // of the lane's column (one without a row: another's numbers, not stored)
        const float* sw;
        float scale;
        int first, count, split, b, hi;
    };
    auto start = [&](int item) {
        Item it;
        const int entry = item / g.splits;
        it.split = item - entry * g.splits;
        it.first = entries[3 * entry + 1];
        it.count = entries[3 * entry + 2];
        it.b = blocks * it.split / g.splits;
        it.hi = blocks * (it.split + 1) / g.splits;
        const int pair = places[it.first + min(gr, it.count - 1)];
        it.row = g.hidden + (size_t)pair * g.F + t4 * (PER / 8) + it.b * PER;
        it.scale = FP8 ? few_scale(largest[pair], HIDDEN_TO) : 1.0f;
        it.sw = FP8 ? g.s_out + ((size_t)entries[3 * entry] * db + min(n0, g.D - 1) / 128) * fb : nullptr;
        return it;
    };
    float4 next[2][HW];
    float s_next = 1.0f;
    auto fetch = [&](Item& it, int b) {
        if (whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < HW; ++i) next[h][i] = *reinterpret_cast<const float4*>(it.row + h * (PER / 2) + i * 4);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < HW; ++i) {
                    const int k = h * (PER / 2) + i * 4;
                    next[h][i] = b * PER + t4 * (PER / 8) + k < g.F ? *reinterpret_cast<const float4*>(it.row + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);      // (F is a multiple of 8)
                }
        }
        it.row += PER;
        if (FP8) s_next = it.sw[b];
    };
    int item = warp, slot = 0;
    Item here, after;
    if (item < items) {
        here = start(item);
        fetch(here, here.b);
    }
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
    while (item < items) {
        // the operand's pairs: two fp16 (the second with its sign turned) or bf16 parts
        uint2 high[2][HW], low[2][HW];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < HW; ++i) {
                const float4 v = next[h][i];
                if (FP8) {
                    const float2 a = times(v.x, v.y, here.scale), b = times(v.z, v.w, here.scale);
                    const uint2 p = make_uint2(pair_f16(a.x, a.y), pair_f16(b.x, b.y));
                    high[h][i] = p;
                    low[h][i] = make_uint2(f16_excess(p.x, a.x, a.y), f16_excess(p.y, b.x, b.y));
                } else {
                    const uint2 p = make_uint2(pair_bf16(v.x, v.y), pair_bf16(v.z, v.w));
                    high[h][i] = p;
                    low[h][i] = make_uint2(pair_bf16(v.x - low_of(p.x), v.y - high_of(p.x)), pair_bf16(v.z - low_of(p.y), v.w - high_of(p.y)));
                }
            }
        const float s0 = s_next;
        const bool last = here.b + 1 == here.hi;
        if (!last) {
            fetch(here, here.b + 1);
        } else if (item + FEW_WARPS < items) {
            after = start(item + FEW_WARPS);
            fetch(after, after.b);
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(FEW_RING - 1) : "memory");
        const unsigned char* at = ring + slot * FEW_SLOT + lane * 16;
        float c[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 wl = *reinterpret_cast<const uint4*>(at + 1024 * h), wh = *reinterpret_cast<const uint4*>(at + 512 + 1024 * h);
            const uint32_t lw[4] = {wl.x, wl.y, wl.z, wl.w}, hw[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
            for (int i = 0; i < HW; ++i) {
                if (FP8) {
                    uint32_t a0, a1, a2, a3;
                    f16_of(lw[i], a0, a2);
                    f16_of(hw[i], a1, a3);
                    mma_f16_f32(c[0], a0, a1, a2, a3, high[h][i].x, high[h][i].y);
                    mma_f16_f32(c[1], a0, a1, a2, a3, low[h][i].x, low[h][i].y);
                } else {
                    mma_bf16_f32(c[0], lw[2 * i], hw[2 * i], lw[2 * i + 1], hw[2 * i + 1], high[h][i].x, high[h][i].y);
                    mma_bf16_f32(c[1], lw[2 * i], hw[2 * i], lw[2 * i + 1], hw[2 * i + 1], low[h][i].x, low[h][i].y);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = FP8 ? fmaf(s0, c[0][i] - c[1][i], acc[i]) : acc[i] + (c[0][i] + c[1][i]);
        load(slot);
        few_commit();
        slot = slot + 1 == FEW_RING ? 0 : slot + 1;
        if (last) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = t4 * 2 + j;
                if (col < here.count) {
                    const int pair = places[here.first + col];
                    const float back = FP8 ? few_unscale(largest[pair], HIDDEN_TO) : 1.0f;
                    float* to = sums + ((size_t)here.split * pairs + pair) * 16 + gr;
                    to[0] = acc[j] * back;
                    to[8] = acc[2 + j] * back;
                }
                acc[j] = acc[2 + j] = 0.0f;
            }
            here = after;
            item += FEW_WARPS;
        } else {
            ++here.b;
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
    return (size_t)FEW_WARPS * FEW_RING * FEW_SLOT + 4 * ((size_t)(g.s_in ? 2 : 1) * FEW_WARPS * 16 * 16 + few_list_words(g.n, g.E, g.n * g.top));
}
size_t out_smem(const FewArgs& g) {
    const int pairs = g.n * g.top;
    return (size_t)FEW_WARPS * FEW_RING * FEW_SLOT + 4 * ((size_t)g.splits * pairs * 16 + 6 * pairs);
}

constexpr size_t FEW_SMEM = 227 * 1024;

template <bool FP8, bool XS>
int launch(FewArgs& g, cudaStream_t s) {
    constexpr size_t most = FEW_SMEM;
    const size_t smem_in = in_smem(g) + (XS ? (size_t)g.n * few_x_bytes(g.D, FP8) : 0), smem_out = out_smem(g);
    MM_REQUIRE(smem_in <= most && smem_out <= most, "moe few: too many experts or choices for the kernels' shared memory");
    if (!mm_allow_smem<few_in_kernel<FP8, XS>>(most) || !mm_allow_smem<few_out_kernel<FP8>>(most)) {
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
    static std::atomic<int> resident{0};          // (asked for the most shared memory, so that no call's sizes decide for the next)
    int fit = resident.load(std::memory_order_relaxed);
    if (fit == 0) {
        cfg.gridDim = dim3(FP8_SM_COUNT / FEW_CLUSTER * FEW_CLUSTER);
        cfg.dynamicSmemBytes = most;
        if (cudaOccupancyMaxActiveClusters(&fit, few_in_kernel<FP8, XS>, &cfg) != cudaSuccess || fit < 1) {
            (void)cudaGetLastError();
            fit = FEW_CLUSTERS;
        }
        if (fit > FEW_CLUSTERS) fit = FEW_CLUSTERS;
        resident.store(fit, std::memory_order_relaxed);
        cfg.dynamicSmemBytes = smem_in;
    }
    const int most_experts = g.E < g.n * g.top ? g.E : g.n * g.top;
    const long long groups = ((long long)most_experts * (g.F / 8) * g.KS + FEW_WARPS - 1) / FEW_WARPS, clusters = (groups + FEW_CLUSTER - 1) / FEW_CLUSTER;
    cfg.gridDim = dim3((unsigned)(clusters < fit ? clusters : fit) * FEW_CLUSTER);
    cudaLaunchKernelEx(&cfg, few_in_kernel<FP8, XS>, g);
    MM_CHECK_LAUNCH();
    mm_launch_dependent(g_mm_pdl != 0, few_out_kernel<FP8>, dim3(ceil_div(g.D, 16)), dim3(FEW_THREADS), smem_out, s, g);
    MM_CHECK_LAUNCH();
    return MM_OK;
}

}  // namespace

// x bf16 [n, ldx]; w_router fp32 [E, D]; experts bf16 (s_in, s_out null): w_in [E, 2 F, D] (gate rows then up rows, or with `interleaved` alternating in
// blocks of 8), w_out [E, D, F]; or e4m3 with scales: w_in [E, 2, F, ld_in], w_out [E, D, ld_out].  ld_in, ld_out: bytes of a row.
// out bf16 [n, D].  scratch: pairs * (4 F + F / 2 + 24) + 32 + 36 n (D + 160) bytes, pairs = n * top.
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
    g.x_copy = (uint8_t*)(((uintptr_t)(g.lists + 1 + 4 * pairs) + 15) & ~(uintptr_t)15);
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
    const bool xs = in_smem(g) + (size_t)n * few_x_bytes(D, fp8) <= FEW_SMEM;
    if (fp8) return xs ? launch<true, true>(g, s) : launch<true, false>(g, s);
    return xs ? launch<false, true>(g, s) : launch<false, false>(g, s);
}
