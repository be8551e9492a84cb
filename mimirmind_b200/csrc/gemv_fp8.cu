// Products of up to 16 rows with weights in 8 bits (fp8.cuh): the weights are streamed once, from memory into registers.
//
// mma.sync m16n8k32 on e4m3: 16 weight rows are the 16-row operand, the rows of x (padded to 8 or 16) the 8 columns.  The order of k inside a
// block of 128 is free as long as both operands agree, so a lane takes 16 consecutive bytes of a weight row straight from memory and the same of
// x.  A block's four products start from nought; their results are multiplied by the block's scales and added up in fp32.
//
// A CTA's eight warps are RT tiles of 16 rows times KS runs of blocks.  Every warp keeps three blocks on their way (asynchronous copies, over
// tile borders too: 96 KB of weights an SM); a lane copies just the bytes that it reads itself, so no lane waits for another.  The runs' sums
// meet in shared memory and are added in order, so a result does not depend on what runs beside it.
//
// GLU: a tile is 8 rows of the gate's matrix and the same 8 of the up projection's.  A cluster of S CTAs makes the 128 columns of
// one block of the hidden rows, finds the largest number over distributed shared memory and writes the block quantised: the next product reads it as it is.
//
// Few rows are quantised here (every warp its own run of blocks, into shared memory) instead of by a launch of their own in front of this one.
//
// Bound by memory where the matrix is large: 1 x 152,064 x 3,584 84 to 87 us (6.2 TB/s of 6.55).  Smaller ones by the launch, the first block's way from memory and the
// ends of the runs: 8 x 18,944 x 3,584 12.7 us (68 MB, floor 10.4), 8 x 4,608 x 3,584 5.9 us (16.5 MB, floor 2.5).  Four blocks on their way
// instead of three were no faster; a ring in registers instead of shared memory spilled.
#include "fp8.cuh"
#include "fp8_launch.h"

namespace {

constexpr int GV_THREADS = 256, GV_WARPS = 8, RING = 3;
constexpr int GV_MAX_SMEM = 113 * 1024;       // two CTAs an SM

struct GemvArgs {
    const void* x;              // QUANT: the rows, bf16 or fp32
    const uint8_t* q;           // else: e4m3 [m, ldq]
    const float* sa;            // [m, KB]
    const uint8_t* W;
    const float* sw;
    const void* bias;
    void* out;                  // [m, ldo] bf16 or fp32; GLU: e4m3
    float* out_scales;          // GLU: [m, NB]
    long long ldx, ldq, ldw;
    int x_dtype, bias_dtype, out_dtype, act;
    float limit;
    int m, N, K, KB, NB, ldo, RT, KS, S, tiles;
};

// 16 bytes of a row of K from k on, noughts behind its end (nothing there is read): on their way to shared memory, or into registers
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, int k, int K) {      // src = row + k
    const int n = min(max(K - k, 0), 16);
    if (n == 0) src -= k;
    asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ uint4 load16(const uint8_t* row, int k, int K) {
    if (k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < K) w[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void mma_e4m3(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A slot of a warp's ring: a block of its tile's 16 rows (a lane's four pieces: bytes t * 16 .. + 15 and 64 on of rows g and g + 8).
constexpr int SLOT = 2048;
__host__ __device__ inline int q_stride(int KB) { return KB * FP8_BLOCK + 64; }      // 64: rows of neighbouring lanes in different banks

template <int G, bool GLU, bool QUANT>
__global__ void __launch_bounds__(GV_THREADS, 2) gemv_fp8_kernel(const __grid_constant__ GemvArgs g) {
    constexpr int TOK = 8 * G;
    extern __shared__ __align__(16) unsigned char gv_smem[];
    float* part = reinterpret_cast<float*>(gv_smem + GV_WARPS * RING * SLOT);              // [2][8 warps][16 rows][TOK]
    float* hidden = part + 2 * GV_WARPS * 16 * TOK;                                        // GLU: [TOK][128 / S]
    uint32_t* largest = reinterpret_cast<uint32_t*>(hidden + (GLU ? TOK * 128 : 0));      // GLU: [TOK]
    float* x_scales = reinterpret_cast<float*>(largest + (GLU ? TOK : 0));                // [m][KB]
    uint8_t* q_rows = reinterpret_cast<uint8_t*>(x_scales + ((g.m * g.KB + 3) & ~3));     // QUANT: [m][q_stride]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t4 = lane & 3;
    const int ks = warp % g.KS, rt = warp / g.KS;
    const int lo = g.KB * ks / g.KS, hi = g.KB * (ks + 1) / g.KS, nb = hi - lo;
    const int rank = GLU ? blockIdx.x % g.S : 0, first = GLU ? blockIdx.x / g.S : blockIdx.x;
    // steps of RT tiles each: the plain form walks over the matrix, a GLU CTA over its share of one block's sixteen tiles
    const int steps = GLU ? 16 / g.S / g.RT : (g.tiles - first * g.RT + (int)gridDim.x * g.RT - 1) / ((int)gridDim.x * g.RT);
    unsigned char* ring = gv_smem + warp * RING * SLOT;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;

    // the cursor of loading: the run's next block, over the steps
    const int total = nb * steps;
    const bool whole = g.K % FP8_BLOCK == 0;
    int load_step = 0, load_b = lo;
    const uint8_t *pa, *pb;
    auto first_row = [&](int step) {
        return GLU ? first * 128 + (rank * (16 / g.S) + step * g.RT + rt) * 8 : ((first + step * (int)gridDim.x) * g.RT + rt) * 16;
    };
    auto point = [&]() {
        const int n0 = first_row(load_step), ra = min(n0 + gr, g.N - 1), rb = GLU ? g.N + ra : min(n0 + gr + 8, g.N - 1);
        const int k = lo * FP8_BLOCK + t4 * 16;
        pa = g.W + (size_t)ra * g.ldw + k;
        pb = g.W + (size_t)rb * g.ldw + k;
    };
    point();
    auto load_weights = [&](int slot) {
        const uint32_t dst = ring_at + slot * SLOT;
        if (whole) {
            copy16(dst, pa);
            copy16(dst + 512, pb);
            copy16(dst + 1024, pa + 64);
            copy16(dst + 1536, pb + 64);
        } else {
            const int k = load_b * FP8_BLOCK + t4 * 16;
            copy16(dst, pa, k, g.K);
            copy16(dst + 512, pb, k, g.K);
            copy16(dst + 1024, pa + 64, k + 64, g.K);
            copy16(dst + 1536, pb + 64, k + 64, g.K);
        }
        pa += FP8_BLOCK;
        pb += FP8_BLOCK;
        if (++load_b == hi) {
            load_b = lo;
            ++load_step;
            point();
        }
    };
    // the same block of x, a block ahead in registers (a warp's block takes longer than a load from L2)
    uint4 next[G][2];
    const uint8_t* rows[G];
#pragma unroll
    for (int j = 0; j < G; ++j) rows[j] = QUANT ? q_rows + (size_t)min(j * 8 + gr, g.m - 1) * q_stride(g.KB) : g.q + (size_t)min(j * 8 + gr, g.m - 1) * g.ldq;
    auto load_rows = [&](int b) {
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int tok = j * 8 + gr;
                const int k = b * FP8_BLOCK + t4 * 16 + 64 * h;
                if (tok >= g.m) next[j][h] = make_uint4(0, 0, 0, 0);
                else if (whole) next[j][h] = *reinterpret_cast<const uint4*>(rows[j] + k);
                else next[j][h] = load16(rows[j], k, g.K);
            }
    };
#pragma unroll 1
    for (int i = 0; i < RING; ++i) {
        if (i < total) load_weights(i);      // weights do not depend on the launch before
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!QUANT) load_rows(lo);

    if (QUANT) {
        // half a warp per (row, block), eight numbers a lane
        const bool wide = g.K % 8 == 0 && g.ldx % 8 == 0 && ((uintptr_t)g.x & 15) == 0;
        const int hl = lane & 15, units = g.m * g.KB;
        for (int u0 = warp * 2; u0 < units; u0 += 2 * GV_WARPS) {
            const int u = u0 + (lane >> 4), row = u / g.KB, b = u - row * g.KB, k = b * FP8_BLOCK + hl * 8;
            const bool on = u < units;
            float v[8];
            if (on && wide && k + 8 <= g.K) {
                if (g.x_dtype == MM_F32) fp8_load8<float>((const float*)g.x + (size_t)row * g.ldx + k, v);
                else fp8_load8<__nv_bfloat16>((const __nv_bfloat16*)g.x + (size_t)row * g.ldx + k, v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = !on || k + i >= g.K ? 0.0f
                           : g.x_dtype == MM_F32 ? ((const float*)g.x)[(size_t)row * g.ldx + k + i]
                                                 : __bfloat162float(((const __nv_bfloat16*)g.x)[(size_t)row * g.ldx + k + i]);
            }
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) big = max(big, fp8_size_bits(v[i]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
            const float s = fp8_scale_of(big);
            fp8_quotients<8>(v, s);
            if (on) {
                if (hl == 0) x_scales[row * g.KB + b] = s;
                *reinterpret_cast<uint2*>(q_rows + (size_t)row * q_stride(g.KB) + k) = make_uint2(fp8_pack4(v[0], v[1], v[2], v[3]), fp8_pack4(v[4], v[5], v[6], v[7]));
            }
        }
    } else {
        for (int i = threadIdx.x; i < g.m * g.KB; i += GV_THREADS) x_scales[i] = g.sa[i];
    }
    __syncthreads();
    float acc[G][4];
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;

    int done = 0, slot = 0;
    const float *xa[G], *xb[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
        xa[j] = x_scales + min(j * 8 + t4 * 2, g.m - 1) * g.KB;
        xb[j] = x_scales + min(j * 8 + t4 * 2 + 1, g.m - 1) * g.KB;
    }
    for (int step = 0; step < steps; ++step) {
        const float* sw = g.sw + (size_t)(min(first_row(step), g.N - 1) / FP8_BLOCK) * g.KB;      // (read a block ahead)
        const float* su = sw + (size_t)g.NB * g.KB;
        float s0_next = sw[lo], s1_next = GLU ? su[lo] : 0.0f;
#pragma unroll 1
        for (int b = lo; b < hi; ++b) {
            uint4 now[G][2];
            if (!QUANT) {
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    now[j][0] = next[j][0];
                    now[j][1] = next[j][1];
                }
                load_rows(b + 1 < hi ? b + 1 : lo);
            }
            asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");       // this lane's oldest copies have landed
            const unsigned char* at = ring + slot * SLOT + lane * 16;
            uint4 wl[2], wh[2];
            wl[0] = *reinterpret_cast<const uint4*>(at);
            wh[0] = *reinterpret_cast<const uint4*>(at + 512);
            wl[1] = *reinterpret_cast<const uint4*>(at + 1024);
            wh[1] = *reinterpret_cast<const uint4*>(at + 1536);
            const float s0 = s0_next, s1 = GLU ? s1_next : s0;
            if (b + 1 < hi) {
                s0_next = sw[b + 1];
                if (GLU) s1_next = su[b + 1];
            }
#pragma unroll
            for (int j = 0; j < G; ++j) {
                uint4 x[2];
                if (QUANT) {
                    const uint8_t* row = rows[j] + b * FP8_BLOCK + t4 * 16;
                    x[0] = *reinterpret_cast<const uint4*>(row);
                    x[1] = *reinterpret_cast<const uint4*>(row + 64);
                } else {
                    x[0] = now[j][0];
                    x[1] = now[j][1];
                }
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mma_e4m3(c, wl[h].x, wh[h].x, wl[h].y, wh[h].y, x[h].x, x[h].y);
                    mma_e4m3(c, wl[h].z, wh[h].z, wl[h].w, wh[h].w, x[h].z, x[h].w);
                }
                const float sa = xa[j][b], sb = xb[j][b];
                acc[j][0] = fmaf(sa * s0, c[0], acc[j][0]);
                acc[j][1] = fmaf(sb * s0, c[1], acc[j][1]);
                acc[j][2] = fmaf(sa * s1, c[2], acc[j][2]);
                acc[j][3] = fmaf(sb * s1, c[3], acc[j][3]);
            }
            // the slot's numbers have been multiplied: the run's next block but three goes there
            if (done + RING < total) load_weights(slot);
            asm volatile("cp.async.commit_group;" ::: "memory");
            ++done;
            slot = slot + 1 == RING ? 0 : slot + 1;
        }
        float* mine = part + (((step & 1) * GV_WARPS + warp) * 16 + gr) * TOK + t4 * 2;
#pragma unroll
        for (int j = 0; j < G; ++j) {
            *reinterpret_cast<float2*>(mine + j * 8) = make_float2(acc[j][0], acc[j][1]);
            *reinterpret_cast<float2*>(mine + 8 * TOK + j * 8) = make_float2(acc[j][2], acc[j][3]);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
        }
        __syncthreads();
        const float* all = part + (step & 1) * GV_WARPS * 16 * TOK;
        const int rows = GLU ? 8 * g.RT : 16 * g.RT, items = rows * g.m;
        for (int i = threadIdx.x; i < items; i += GV_THREADS) {
            const int tok = i / rows, r = i % rows, tile = GLU ? r >> 3 : r >> 4, row = GLU ? r & 7 : r & 15;
            const float* p = all + (tile * g.KS * 16 + row) * TOK + tok;
            float y = 0.0f, u = 0.0f;
            for (int s = 0; s < g.KS; ++s) {
                y += p[s * 16 * TOK];
                if (GLU) u += p[s * 16 * TOK + 8 * TOK];
            }
            if (GLU) {
                const int col = step * g.RT * 8 + r, f = first * 128 + rank * (128 / g.S) + col;
                hidden[tok * (128 / g.S) + col] = f < g.N ? fp8_glu(y, u, g.act, g.limit, 1.0f) : 0.0f;
            } else {
                const int n = (first + step * (int)gridDim.x) * g.RT * 16 + r;
                if (n < g.N) {
                    if (g.bias) y += g.bias_dtype == MM_F32 ? ((const float*)g.bias)[n] : __bfloat162float(((const __nv_bfloat16*)g.bias)[n]);
                    if (g.out_dtype == MM_F32) ((float*)g.out)[(size_t)tok * g.ldo + n] = y;
                    else ((__nv_bfloat16*)g.out)[(size_t)tok * g.ldo + n] = __float2bfloat16_rn(y);
                }
            }
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (GLU) {
        // a warp per row of x: the largest of this CTA's columns, then of the cluster's, then the quotients
        const int cols = 128 / g.S;
        __syncthreads();
        for (int tok = warp; tok < g.m; tok += GV_WARPS) {
            uint32_t big = 0;
            for (int c = lane; c < cols; c += 32) big = max(big, fp8_size_bits(hidden[tok * cols + c]));
            big = __reduce_max_sync(0xffffffffu, big);
            if (lane == 0) largest[tok] = big;
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int tok = warp; tok < g.m; tok += GV_WARPS) {
            uint32_t big = 0;
            for (int r = 0; r < g.S; ++r) {
                uint32_t at = (uint32_t)__cvta_generic_to_shared(largest + tok), v;
                asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(r));
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
                big = max(big, v);
            }
            const float s = fp8_scale_of(big);
            if (rank == 0 && lane == 0) g.out_scales[(size_t)tok * g.NB + first] = s;
            const int c = lane * 4, f = first * 128 + rank * cols + c;
            if (c < cols && f < g.ldo) {
                const float* from = hidden + tok * cols + c;
                float h[4] = {from[0], from[1], from[2], from[3]};
                fp8_quotients<4>(h, s);
                *reinterpret_cast<uint32_t*>((uint8_t*)g.out + (size_t)tok * g.ldo + f) = fp8_pack4(h[0], h[1], h[2], h[3]);
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // nobody leaves while another may read its shared memory
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

template <int G, bool GLU, bool QUANT>
int launch(const GemvArgs& g, int grid, size_t smem, bool dependent, cudaStream_t s) {
    if (smem > 48 * 1024 && !mm_allow_smem<gemv_fp8_kernel<G, GLU, QUANT>>(GV_MAX_SMEM)) {
        mm_set_last_error("gemv_fp8: cannot reserve shared memory");
        return MM_ERR_LAUNCH;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(GV_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (GLU) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = g.S;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent && g_mm_pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaLaunchKernelEx(&cfg, gemv_fp8_kernel<G, GLU, QUANT>, g);
    MM_CHECK_LAUNCH();
    return MM_OK;
}

}  // namespace

static size_t gemv_smem(int m, int KB, bool glu, bool quant) {
    const int tok = m <= 8 ? 8 : 16;
    return (size_t)GV_WARPS * RING * SLOT + (size_t)2 * GV_WARPS * 16 * tok * 4 + (glu ? (size_t)tok * 128 * 4 + tok * 4 : 0) +
           (size_t)((m * KB + 3) & ~3) * 4 + (quant ? (size_t)m * q_stride(KB) : 0);
}

bool fp8_gemv_takes(int m, int K, bool glu, bool quant) {
    return m <= 16 && K < (1 << 20) && gemv_smem(m, ceil_div(K, FP8_BLOCK), glu, quant) <= GV_MAX_SMEM;
}

int fp8_gemv(const Fp8In& x, const Fp8Mat& w, const Fp8Out& out, bool glu, bool dependent, cudaStream_t s) {
    GemvArgs g = {};
    const bool quant = x.dtype != FP8_QUANTISED;
    g.x = x.data;
    g.q = (const uint8_t*)x.data;
    g.sa = x.scales;
    g.ldx = x.ld;
    g.ldq = x.ld;
    g.x_dtype = x.dtype;
    g.W = (const uint8_t*)w.values;
    g.sw = w.scales;
    g.ldw = w.ld;
    g.bias = out.bias;
    g.bias_dtype = out.bias_dtype;
    g.out = out.data;
    g.out_dtype = out.dtype;
    g.out_scales = out.scales;
    g.ldo = out.ld;
    g.act = out.act;
    g.limit = out.limit;
    g.m = x.rows;
    g.N = w.N;
    g.K = w.K;
    g.KB = ceil_div(w.K, FP8_BLOCK);
    g.NB = ceil_div(w.N, FP8_BLOCK);
    g.tiles = ceil_div(w.N, 16);
    // Tiles side by side in a CTA (8, 4, 2, 1) and runs of blocks (no more than blocks): the least number of blocks that a warp goes through one after the other, a meeting
    // of the warps counted as one, and less than one and a half CTAs an SM as that much less bandwidth.  Us of 8, 4, 2 and 1 tiles: one row of 27,648 x 5,120 28.8, 31.2,
    // 26.5, 27.1; 65,536 x 3,584 44.2, 43.9, 40.1, 43.7; 32,768 x 1,024 9.8, 10.5, 11.4, 12.1; 18,944 x 3,584 17.2, 14.8, 14.6, 15.5; eight rows of 152,064 x 3,584 99, 94, 92, 96.
    int grid;
    if (glu) {
        g.S = 1;
        while (g.S < 8 && g.NB * g.S * 2 <= 2 * FP8_SM_COUNT) g.S *= 2;
        g.RT = g.S == 1 ? GV_WARPS : 16 / g.S;
        while (GV_WARPS / g.RT > g.KB) {
            if (16 / g.S < g.RT * 2) g.S /= 2;
            g.RT *= 2;
        }
        grid = g.NB * g.S;
    } else {
        float best = 1e30f;
        for (int rt = GV_WARPS; rt >= 1 && GV_WARPS / rt <= g.KB; rt /= 2) {
            const int n = ceil_div(g.tiles, rt);
            const float cost = (float)ceil_div(n, 2 * FP8_SM_COUNT) * ((float)g.KB * rt / GV_WARPS + 1.0f) * (n < FP8_SM_COUNT * 3 / 2 ? FP8_SM_COUNT * 1.5f / n : 1.0f);
            if (cost < best) {
                best = cost;
                g.RT = rt;
            }
        }
        const int groups = ceil_div(g.tiles, g.RT);
        grid = groups < 2 * FP8_SM_COUNT ? groups : 2 * FP8_SM_COUNT;
    }
    g.KS = GV_WARPS / g.RT;
    const int G = g.m <= 8 ? 1 : 2;
    const size_t smem = gemv_smem(g.m, g.KB, glu, quant);
    MM_REQUIRE(smem <= GV_MAX_SMEM, "gemv_fp8: rows too long for the kernel's shared memory");
    if (glu) {
        if (quant) return G == 1 ? launch<1, true, true>(g, grid, smem, dependent, s) : launch<2, true, true>(g, grid, smem, dependent, s);
        return G == 1 ? launch<1, true, false>(g, grid, smem, dependent, s) : launch<2, true, false>(g, grid, smem, dependent, s);
    }
    if (quant) return G == 1 ? launch<1, false, true>(g, grid, smem, dependent, s) : launch<2, false, true>(g, grid, smem, dependent, s);
    return G == 1 ? launch<1, false, false>(g, grid, smem, dependent, s) : launch<2, false, false>(g, grid, smem, dependent, s);
}
