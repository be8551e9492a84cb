// Products of rows and weights in 8 bits on the fifth-generation tensor cores, with a scale per row and block of 128 and per weight
// block of 128 x 128 (fp8.cuh):
//   y[m, n] = sum over blocks b of sa[m, b] sw[n / 128, b] (sum over k in b of qa[m, k] qw[n, k])  (+ bias[n]).
//
// tcgen05.mma kind::f8f6f4 (128 x BN x 32, fp32 in tensor memory) makes one block's inner sums from operands that TMA brought into shared
// memory (rows of 128 bytes, 128-byte swizzle); while it makes the next block's, eight warps read these back, multiply them by the block's
// scales and add them to sums in registers, BN / 2 columns of one row a thread, with two accumulators in tensor memory, one per block in turn.
//
// Roles: warps 0..7 sums and results, warps 8 and 11 TMA, warps 9 and 10 products, each of the two for every other block (one thread that issued for all
// took 960 cycles a block).  A block of a 128 x 256 tile is 512 cycles of the tensor pipe.  What bounds the loop is the round of an accumulator, 1,620 cycles, in which
// every one of the two makes a block, 810 a block: from issue to the end of its products 600, the wait for
// them 200, reading 470, the next products' issue 350.  Pairs of CTAs (cta_group::2, 256 rows a tile, a third less traffic in shared memory) have
// the same round, with or without the tile in halves, and were not faster (4,096 x 18,944 x 3,584: 281 and 295 us against 272); halves of one CTA's tile, each
// 128 columns with barriers of its own, took 410; weights fetched into L2 8 to 24 blocks ahead 278.  A tile's end (results through shared memory in rows of 128 bytes;
// GLU: the exponentials and quotients) takes 3,000 to 5,000 cycles, its start 1,400.  A CTA walks over tiles, row tiles first, so that CTAs at work at
// the same time share weight tiles in L2.  Few tiles: a cluster of S CTAs splits a tile's blocks; every CTA puts its sums into its own shared
// memory, and after a cluster barrier each finishes every S-th row from all S in rank order (the same order on every run).
//
// Kinds of result: rows in bf16 or fp32 (+ bias); or, GLU, W holds pairs of matrices (the gate's and the up projection's), a tile is 128 columns of
// both, and act(gate, up) leaves as e4m3 rows with their scales: the 128 columns are one block of the next product's rows, so its largest
// number is known here and the hidden rows never exist in another form.
//
// Grouped form: row tiles of a device-made list (first row, end row, matrix), as in gemm_tcgen05.cu.
//
// Measured, rows quantised before: 4,096 x 18,944 x 3,584 257 us (2.16 PFLOP/s; under the power cap of a long run 296), 2,000 rows of 5,120 and 2 x 13,824 302, 48 x 3,584 x 3,584 8.5 (12.8 MB,
// 4 CTAs a tile), 333 x 19,001 x 912 29, 11 of which are the odd rows' number by number (whole words, shifted by a number where a row starts at an odd one, were no faster).
//
// Every wait is bounded; when one runs out, the CTA's tiles from there on become NaN, copies in flight get time to land, `err` is set.
#include "fp8.cuh"
#include "fp8_launch.h"
#include "tcgen05.cuh"

namespace {

using namespace tc;

constexpr int T_ROWS = 128, T_THREADS = 384, SUM_WARPS = 8;
constexpr int PIECE = 32;                                        // columns that a summing warp has on their way from tensor memory
// A summing thread of a 256-column tile holds 128 sums and two pieces: registers move from the last warpgroup to the others.
// 256 x 224 + 128 x 56 = 256 x 232 + 128 x 40 = 384 x 168, what the block starts with (the launch checks that).  Sixteen summing warps of half the columns, which 112
// registers each allow, were slower (2,048 x 4,736 x 13,824: 218 us against 178).
constexpr int START_REGS = 168;
__host__ __device__ constexpr int sum_regs(bool glu) { return glu ? 232 : 224; }
__host__ __device__ constexpr int other_regs(bool glu) { return glu ? 40 : 56; }
static_assert(SUM_WARPS * 32 * sum_regs(false) + 128 * other_regs(false) <= T_THREADS * START_REGS &&
              SUM_WARPS * 32 * sum_regs(true) + 128 * other_regs(true) <= T_THREADS * START_REGS, "registers");
constexpr int HALF_BYTES = 128 * 128;              // 128 rows of 128 bytes
enum { OUT_BF16 = 0, OUT_F32 = 1 };

struct Fp8Args {
    void* out;                  // rows, or (GLU) the hidden rows' e4m3 numbers
    float* out_scales;          // (GLU) [M, NB]
    const float* sa;            // [M, KB]
    const float* sw;            // [matrices, NB, KB]
    const void* bias;
    const float* row_scale;     // (GLU) [.] fp32 or null: gate and up sums of row r are multiplied by row_scale[order ? order[r] : r]
    const int32_t* order;
    const int32_t* tiles;       // grouped: 3 ints a row tile
    const int32_t* n_tiles;
    int* err;
    int out_kind, bias_dtype, act;
    float limit;
    int M, N, K, KB, NB, ldo, S;
    int t0, t1;                 // the tiles that this launch makes (grouped: up to the list's end)
};

template <int BN>
struct Layout {
    static constexpr int STAGE_BYTES = HALF_BYTES * (1 + BN / 128);
    static constexpr int STAGES = BN == 256 ? 4 : 6;
    static constexpr int PIPE_BYTES = STAGES * STAGE_BYTES;
    static constexpr int STAGING = 4096;           // per warp: 32 rows of 128 bytes
    static constexpr int PART_LD = BN + 4;         // floats of a row of a split tile's sums
};

struct Ctl {
    uint64_t full[6], empty[6];
    uint64_t sum_full[2], sum_empty[2];
    uint64_t row_known[4];                         // the two warps that hold a row's parts (GLU)
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(128 * Layout<256>::PART_LD * 4 <= Layout<256>::PIPE_BYTES && 128 * Layout<128>::PART_LD * 4 <= Layout<128>::PIPE_BYTES, "split sums");

// fp32 accumulate, e4m3 x e4m3, both K-major, M = 128
__host__ __device__ constexpr uint32_t idesc_e4m3(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(T_ROWS >> 4) << 24); }

__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0) : "memory");
}

// a tensor-memory load on its way, and the wait for it (and all earlier ones of the warp): the values may only be used behind it
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
// the same as a wait, without the instruction: for a second load that the wait before covers
__device__ __forceinline__ void tmem_arrived32(uint32_t* r) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
// two sums in one instruction: (a, b) += s (x, y), s = (s, s)
__device__ __forceinline__ void fma_pair(uint64_t& ab, uint64_t s, uint32_t x, uint32_t y) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(ab) : "l"(((uint64_t)y << 32) | x), "l"(s));
}
__device__ __forceinline__ uint64_t twice(float s) { return ((uint64_t)__float_as_uint(s) << 32) | __float_as_uint(s); }

// mbar_wait for the warps that copy and issue: they sleep on the barrier, a microsecond at the most, instead of asking it time and again beside the summing
// warps (4,096 x 18,944 x 3,584 under the power cap 301 us, so 296; the summing warps themselves lose by it, 306).  Bounded all the same: under 3 s.
__device__ __forceinline__ bool mbar_sleep(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (uint32_t it = 0; it < (1u << 21); ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
        if (ok) return true;
        if ((it & 255u) == 255u && *abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}

__device__ __forceinline__ float bias_at(const Fp8Args& g, int n) {
    return g.bias_dtype == MM_F32 ? ((const float*)g.bias)[n] : __bfloat162float(((const __nv_bfloat16*)g.bias)[n]);
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// A tile: rows lo .. hi - 1 (of one group), first column of the result, first rows of W's two boxes, the scales' rows of W.
struct Tile {
    int m0, hi, n0, w0, w1;
    const float *s0, *s1;
};
template <int BN, bool GLU>
__device__ __forceinline__ Tile tile_of(const Fp8Args& g, int t, int m_tiles) {
    Tile x;
    const int mt = t % m_tiles, nt = t / m_tiles;
    int e = 0;
    if (g.tiles != nullptr) {
        x.m0 = g.tiles[3 * mt];
        x.hi = g.tiles[3 * mt + 1];
        e = g.tiles[3 * mt + 2];
    } else {
        x.m0 = mt * T_ROWS;
        x.hi = g.M;
    }
    if (GLU) {
        x.n0 = nt * 128;
        x.w0 = 2 * e * g.N + x.n0;
        x.w1 = x.w0 + g.N;
        x.s0 = g.sw + ((size_t)2 * e * g.NB + nt) * g.KB;
        x.s1 = x.s0 + (size_t)g.NB * g.KB;
    } else {
        x.n0 = nt * BN;
        x.w0 = e * g.N + x.n0;
        x.w1 = x.w0 + 128;
        const int nb = x.n0 / FP8_BLOCK;
        x.s0 = g.sw + ((size_t)e * g.NB + nb) * g.KB;
        x.s1 = g.sw + ((size_t)e * g.NB + min(nb + 1, g.NB - 1)) * g.KB;      // (columns from N on are not stored)
    }
    return x;
}

// acc[i] = act(acc[i], acc[N + i]): one kind of activation a loop, so that its exponentials and quotients overlap (with the choice inside, a tile's
// end took 10,000 cycles)
template <int ACT, int N>
__device__ __forceinline__ void gated_half(float* acc, float rs, float limit) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fp8_glu_as<ACT>(acc[i], acc[N + i], limit, rs);
}

// 128 bytes of 32 rows on their way to memory: 16-byte unit u of row r at u ^ (r & 7), so that neither side meets bank conflicts
__device__ __forceinline__ unsigned char* staged(unsigned char* base, int r, int u) { return base + r * 128 + ((u ^ (r & 7)) << 4); }

template <typename T>
__device__ __forceinline__ void store_staged(unsigned char* base, int lane, T* out, int ldo, int row0, int hi, int col0, int N, bool wide) {
    constexpr int PER = 128 / sizeof(T), UNIT = 16 / sizeof(T);
    __syncwarp();
    if (wide && col0 + PER <= N) {
        const int r0 = lane >> 3, u = lane & 7;
        T* to = out + (size_t)(row0 + r0) * ldo + col0 + u * UNIT;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (row0 + r0 + i * 4 < hi) *reinterpret_cast<uint4*>(to + (size_t)(i * 4) * ldo) = *reinterpret_cast<const uint4*>(staged(base, r0 + i * 4, u));
    } else {          // rows that start anywhere, or columns that end here: number by number, neighbours side by side
#pragma unroll 4
        for (int i = lane; i < 32 * PER; i += 32) {
            const int r = i / PER, c = i % PER;
            if (row0 + r < hi && col0 + c < N) out[(size_t)(row0 + r) * ldo + col0 + c] = reinterpret_cast<const T*>(staged(base, r, c / UNIT))[c % UNIT];
        }
    }
    __syncwarp();          // the area may be written again
}

template <int BN, bool GLU, bool SPLIT>
__global__ void __launch_bounds__(T_THREADS, 1)
gemm_fp8_tcgen05_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ Fp8Args g) {
    static_assert(!GLU || BN == 256, "a gated tile holds 128 columns of both matrices");
    typedef Layout<BN> L;
    constexpr int COLS = BN / 2, PIECES = COLS / PIECE;      // columns a thread sums
    extern __shared__ unsigned char smem_raw[];
    unsigned char* pipe = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* staging = pipe + L::PIPE_BYTES;
    Ctl* ctl = reinterpret_cast<Ctl*>(staging + SUM_WARPS * L::STAGING);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &ctl->abort_flag;
    // the tile's column of a thread's piece.  GLU: the first half of its sums is of the gate's columns, the second of the up projection's
    auto column = [](int c, int part) { return GLU ? (c < PIECES / 2 ? part * (COLS / 2) + c * PIECE : 128 + part * (COLS / 2) + (c - PIECES / 2) * PIECE) : part * COLS + c * PIECE; };

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmW);
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(smem_u32(&ctl->full[s]), 1);
            mbar_init(smem_u32(&ctl->empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(smem_u32(&ctl->sum_full[a]), 1);
            mbar_init(smem_u32(&ctl->sum_empty[a]), SUM_WARPS);
        }
        for (int q = 0; q < 4; ++q) mbar_init(smem_u32(&ctl->row_known[q]), 2);
        ctl->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == SUM_WARPS + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)), "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = ctl->tmem_base;

    const int m_tiles = g.tiles ? *g.n_tiles : (g.M + T_ROWS - 1) / T_ROWS, n_tiles = (g.N + (GLU ? 128 : BN) - 1) / (GLU ? 128 : BN);
    const int total = g.tiles ? m_tiles * n_tiles : g.t1;
    const int S = SPLIT ? g.S : 1, rank = SPLIT ? (int)cluster_ctarank() : 0;
    const int first = g.t0 + (SPLIT ? blockIdx.x / S : blockIdx.x), step = SPLIT ? 0x40000000 : (int)gridDim.x;      // a split tile has its cluster for itself
    const int b_lo = SPLIT ? (int)((long long)g.KB * rank / S) : 0, b_hi = SPLIT ? (int)((long long)g.KB * (rank + 1) / S) : g.KB;

    if (warp >= SUM_WARPS) {
        if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(other_regs(GLU)));
        const int turn = warp >= SUM_WARPS + 2 ? 1 : 0;        // the blocks of even numbers, or of odd ones
        if (warp == SUM_WARPS || warp == SUM_WARPS + 3) {
            if (lane == 0) {
                uint32_t it = 0;
                bool ok = true;
                for (int t = first; t < total && ok; t += step) {
                    const Tile x = tile_of<BN, GLU>(g, t, m_tiles);
                    for (int b = b_lo; b < b_hi; ++b, ++it) {
                        const int s = it % L::STAGES;
                        if ((it & 1) != turn) continue;
                        if (!mbar_sleep(smem_u32(&ctl->empty[s]), ((it / L::STAGES) & 1) ^ 1, abort_flag)) { ok = false; break; }
                        const uint32_t full = smem_u32(&ctl->full[s]), dst = smem_u32(pipe + s * L::STAGE_BYTES);
                        mbar_expect_tx(full, L::STAGE_BYTES);
                        tma_load_2d(dst + HALF_BYTES, &tmW, b * FP8_BLOCK, x.w0, full);
                        if (BN == 256) tma_load_2d(dst + 2 * HALF_BYTES, &tmW, b * FP8_BLOCK, x.w1, full);
                        tma_load_2d(dst, &tmA, b * FP8_BLOCK, x.m0, full);
                    }
                }
            }
        } else {
            if (lane == 0) {
                uint32_t it = 0;
                bool ok = true;
                for (int t = first; t < total && ok; t += step)
                    for (int b = b_lo; b < b_hi; ++b, ++it) {
                        const int s = it % L::STAGES, acc = it & 1;
                        if (acc != turn) continue;
                        const uint32_t a_addr = smem_u32(pipe + s * L::STAGE_BYTES);
                        const uint64_t a_desc = smem_desc_sw128(a_addr, 16, 1024), b_desc = smem_desc_sw128(a_addr + HALF_BYTES, 16, 1024);
                        if (!mbar_sleep(smem_u32(&ctl->full[s]), (it / L::STAGES) & 1, abort_flag) ||
                            !mbar_sleep(smem_u32(&ctl->sum_empty[acc]), ((it >> 1) & 1) ^ 1, abort_flag)) { ok = false; break; }
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < 4; ++k)          // 32 numbers a product: 32 bytes on along the swizzled rows
                            umma_e4m3(tmem_base + acc * BN, a_desc + (uint64_t)(k * 2), b_desc + (uint64_t)(k * 2), idesc_e4m3(BN), k ? 1u : 0u);
                        umma_commit(smem_u32(&ctl->empty[s]));          // (a commit, not a summing thread's arrival: 263 us against 258)
                        umma_commit(smem_u32(&ctl->sum_full[acc]));
                    }
            }
        }
        if (SPLIT) {
            __syncwarp();
            pair_sync();
        }
    } else {
        if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(sum_regs(GLU)));
        const int q = warp & 3, part = warp >> 2;
        const uint32_t taddr = tmem_base + ((uint32_t)(q * 32) << 16);
        unsigned char* wstage = staging + warp * L::STAGING;
        uint32_t it = 0, known = 0;
        bool ok = true;
        for (int t = first; t < total; t += step) {
            const Tile x = tile_of<BN, GLU>(g, t, m_tiles);
            const int row = x.m0 + q * 32 + lane;
            const float* sa = g.sa + (size_t)min(row, x.hi - 1) * g.KB;
            const float* sw = GLU || BN == 128 || part == 0 ? x.s0 : x.s1;
            uint64_t sums[COLS / 2];
#pragma unroll
            for (int i = 0; i < COLS / 2; ++i) sums[i] = 0;
            float a_next = b_lo < b_hi ? sa[b_lo] : 0.0f, w_next = b_lo < b_hi ? sw[b_lo] : 0.0f, u_next = GLU && b_lo < b_hi ? x.s1[b_lo] : 0.0f;
#pragma unroll 1
            for (int b = b_lo; b < b_hi && ok; ++b, ++it) {
                const uint32_t ph = it & 1;
                const uint64_t s0 = twice(a_next * w_next), s1 = GLU ? twice(a_next * u_next) : 0;
                if (b + 1 < b_hi) {
                    a_next = sa[b + 1];
                    w_next = sw[b + 1];
                    if (GLU) u_next = x.s1[b + 1];
                }
                ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&ctl->sum_full[ph]), (it >> 1) & 1, abort_flag));
                if (!ok) break;
                tc_fence_after();
                // Two pieces are on their way at a time, and the wait is for both: what bounds the loop is how often a warp waits for tensor memory (one
                // piece at a time: 960 cycles a block).  A piece's registers take the next one as soon as they are multiplied; the accumulator is free once the
                // last two have arrived.
                uint32_t r[2][PIECE];
                tmem_ld32_issue(taddr + ph * BN + column(0, part), r[0]);
                tmem_ld32_issue(taddr + ph * BN + column(1, part), r[1]);
#pragma unroll
                for (int c = 0; c < PIECES; c += 2) {
                    tmem_wait32(r[0]);
                    tmem_arrived32(r[1]);
                    if (c + 2 == PIECES) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&ctl->sum_empty[ph]));
                    }
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
#pragma unroll
                        for (int i = 0; i < PIECE; i += 2) fma_pair(sums[((c + d) * PIECE + i) / 2], GLU && c + d >= PIECES / 2 ? s1 : s0, r[d][i], r[d][i + 1]);
                        if (c + 2 < PIECES) tmem_ld32_issue(taddr + ph * BN + column(c + 2 + d, part), r[d]);
                    }
                }
            }
            float acc[COLS];
#pragma unroll
            for (int i = 0; i < COLS / 2; ++i) {
                acc[2 * i] = __uint_as_float((uint32_t)sums[i]);
                acc[2 * i + 1] = __uint_as_float((uint32_t)(sums[i] >> 32));
            }
            if (!ok) {
#pragma unroll
                for (int i = 0; i < COLS; ++i) acc[i] = __uint_as_float(0x7fffffffu);
            }
            if (SPLIT) {
                // this CTA's sums into its own shared memory: the copies have all been read by products that are through
                float* mine = reinterpret_cast<float*>(pipe) + (q * 32 + lane) * L::PART_LD;
                if (row < x.hi) {
#pragma unroll
                    for (int i = 0; i < COLS; i += 4)
                        *reinterpret_cast<float4*>(mine + column(i / PIECE, part) + i % PIECE) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
                }
            } else if (GLU && x.m0 + q * 32 >= x.hi) {
                // none of the tile's rows are this warp's
            } else if (GLU) {
                const float rs = g.row_scale && row < x.hi ? g.row_scale[g.order ? g.order[row] : row] : 1.0f;
                const int n0 = x.n0 + part * (COLS / 2);
                if (g.act == MM_GLU_SILU) gated_half<MM_GLU_SILU, COLS / 2>(acc, rs, g.limit);
                else if (g.act == MM_GLU_CLAMPED) gated_half<MM_GLU_CLAMPED, COLS / 2>(acc, rs, g.limit);
                else gated_half<MM_GLU_GELU_TANH, COLS / 2>(acc, rs, g.limit);
                uint32_t largest = 0;
#pragma unroll
                for (int i = 0; i < COLS / 2; ++i) {
                    if (n0 + i >= g.N) acc[i] = 0.0f;
                    largest = max(largest, fp8_size_bits(acc[i]));
                }
                // the other parts of the row's block are the warps' with the same rows
                volatile uint32_t* sizes = reinterpret_cast<volatile uint32_t*>(staging) + ((known & 1) * 4 + q) * 64 + lane;      // [tile parity][rows' quarter][part][row]
                sizes[part * 32] = largest;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->row_known[q]));
                ok = __all_sync(0xffffffffu, ok && mbar_wait(smem_u32(&ctl->row_known[q]), known & 1, abort_flag));
                ++known;
                const float s = ok ? fp8_scale_of(max(sizes[0], sizes[32])) : __uint_as_float(0x7fffffffu);
                fp8_quotients<COLS / 2>(acc, s);
                if (row < x.hi) {
                    if (part == 0) g.out_scales[(size_t)row * g.NB + x.n0 / 128] = s;
                    uint8_t* dst = (uint8_t*)g.out + (size_t)row * g.ldo + n0;
#pragma unroll
                    for (int i = 0; i < COLS / 2; i += 16) {
                        uint32_t p[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) p[j] = fp8_pack4(acc[i + 4 * j], acc[i + 4 * j + 1], acc[i + 4 * j + 2], acc[i + 4 * j + 3]);
                        if (n0 + i < g.ldo) *reinterpret_cast<uint4*>(dst + i) = make_uint4(p[0], p[1], p[2], p[3]);
                    }
                }
            } else {
                if (g.bias != nullptr) {
#pragma unroll
                    for (int i = 0; i < COLS; ++i)
                        if (x.n0 + part * COLS + i < g.N) acc[i] += bias_at(g, x.n0 + part * COLS + i);
                }
                const bool wide = (((uintptr_t)g.out | ((size_t)g.ldo * (g.out_kind == OUT_F32 ? 4 : 2))) & 15) == 0;
                if (g.out_kind == OUT_F32) {
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            *reinterpret_cast<float4*>(staged(wstage, lane, u)) = make_float4(acc[c + u * 4], acc[c + u * 4 + 1], acc[c + u * 4 + 2], acc[c + u * 4 + 3]);
                        store_staged<float>(wstage, lane, (float*)g.out, g.ldo, x.m0 + q * 32, x.hi, x.n0 + part * COLS + c, g.N, wide);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < COLS; c += 64) {
#pragma unroll
                        for (int u = 0; u < 8; ++u) {
                            uint32_t p[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __nv_bfloat162 v = __floats2bfloat162_rn(acc[c + u * 8 + 2 * j], acc[c + u * 8 + 2 * j + 1]);
                                p[j] = *reinterpret_cast<const uint32_t*>(&v);
                            }
                            *reinterpret_cast<uint4*>(staged(wstage, lane, u)) = make_uint4(p[0], p[1], p[2], p[3]);
                        }
                        store_staged<__nv_bfloat16>(wstage, lane, (__nv_bfloat16*)g.out, g.ldo, x.m0 + q * 32, x.hi, x.n0 + part * COLS + c, g.N, wide);
                    }
                }
            }
        }
        if (SPLIT) {
            __syncwarp();
            pair_sync();               // every CTA's sums stand in its shared memory
            if (first < total) {
                const Tile x = tile_of<BN, GLU>(g, first, m_tiles);
                const uint32_t base = smem_u32(pipe);
                const int rows = min(T_ROWS, x.hi - x.m0);
                for (int r = rank + S * warp; r < rows; r += S * SUM_WARPS) {
                    const int row = x.m0 + r;
                    const float rs = GLU && g.row_scale ? g.row_scale[g.order ? g.order[row] : row] : 1.0f;
                    float4 v[BN / 128];
#pragma unroll
                    for (int j = 0; j < BN / 128; ++j) {
                        const uint32_t at = base + (uint32_t)((r * L::PART_LD + j * 128 + lane * 4) * 4);
                        v[j] = ld_cluster_f4(map_to_rank(at, 0));
                        for (int p = 1; p < S; ++p) {
                            const float4 o = ld_cluster_f4(map_to_rank(at, p));
                            v[j].x += o.x; v[j].y += o.y; v[j].z += o.z; v[j].w += o.w;
                        }
                    }
                    if (GLU) {
                        const float4 ga = v[0], up = v[BN / 128 - 1];
                        const int n = x.n0 + lane * 4;
                        float h[4] = {fp8_glu(ga.x, up.x, g.act, g.limit, rs), fp8_glu(ga.y, up.y, g.act, g.limit, rs),
                                      fp8_glu(ga.z, up.z, g.act, g.limit, rs), fp8_glu(ga.w, up.w, g.act, g.limit, rs)};
                        uint32_t largest = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (n + i >= g.N) h[i] = 0.0f;
                            largest = max(largest, fp8_size_bits(h[i]));
                        }
                        const float s = fp8_scale_of(__reduce_max_sync(0xffffffffu, largest));
                        fp8_quotients<4>(h, s);
                        if (lane == 0) g.out_scales[(size_t)row * g.NB + x.n0 / 128] = s;
                        if (n < g.ldo)
                            *reinterpret_cast<uint32_t*>((uint8_t*)g.out + (size_t)row * g.ldo + n) = fp8_pack4(h[0], h[1], h[2], h[3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < BN / 128; ++j) {
                            const int n = x.n0 + j * 128 + lane * 4;
                            const float y[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (n + i >= g.N) continue;
                                const float z = g.bias ? y[i] + bias_at(g, n + i) : y[i];
                                if (g.out_kind == OUT_F32) ((float*)g.out)[(size_t)row * g.ldo + n + i] = z;
                                else ((__nv_bfloat16*)g.out)[(size_t)row * g.ldo + n + i] = __float2bfloat16_rn(z);
                            }
                        }
                    }
                }
            }
            __syncwarp();
        }
    }

    if (*abort_flag) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    if (SPLIT) pair_sync();        // nobody leaves while another may read its shared memory
    tc_fence_after();
    if (threadIdx.x == 0 && ctl->abort_flag && g.err != nullptr) atomicExch(g.err, 1);
    if (warp == SUM_WARPS + 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN) : "memory");
    }
}

template <int BN, bool GLU, bool SPLIT>
int launch(const CUtensorMap& a, const CUtensorMap& w, const Fp8Args& g, int grid, cudaStream_t s) {
    typedef Layout<BN> L;
    constexpr size_t smem = (size_t)L::PIPE_BYTES + SUM_WARPS * L::STAGING + 1024 + sizeof(Ctl);
    static_assert(smem <= 227 * 1024, "shared memory");
    if (!mm_allow_smem<gemm_fp8_tcgen05_kernel<BN, GLU, SPLIT>>(smem)) {
        mm_set_last_error("gemm_fp8: cannot reserve shared memory");
        return MM_ERR_LAUNCH;
    }
    if (BN == 256) {
        static std::atomic<int> regs{0};          // a register split above what the block starts with would never be granted
        if (regs.load(std::memory_order_relaxed) == 0) {
            cudaFuncAttributes at;
            if (cudaFuncGetAttributes(&at, gemm_fp8_tcgen05_kernel<BN, GLU, SPLIT>) != cudaSuccess) {
                mm_set_last_error("gemm_fp8: cannot read the kernel's attributes");
                return MM_ERR_LAUNCH;
            }
            regs.store(at.numRegs, std::memory_order_relaxed);
        }
        MM_REQUIRE(regs.load(std::memory_order_relaxed) == START_REGS, "gemm_fp8: built with another number of registers than the split wants");
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(T_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = SPLIT ? g.S : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = SPLIT ? 1 : 0;
    cudaLaunchKernelEx(&cfg, gemm_fp8_tcgen05_kernel<BN, GLU, SPLIT>, a, w, g);
    MM_CHECK_LAUNCH();
    return MM_OK;
}

// rows x cols bytes, row stride ld; boxes of 128 x 128, 128-byte swizzle, noughts outside
bool make_map_bytes(CUtensorMap* map, const void* base, long long rows, int cols, long long ld) {
    EncodeTiledFn enc = get_encode();
    if (enc == nullptr) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {128u, 128u};
    cuuint32_t estr[2] = {1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

// tiles t0 .. t1 - 1 (t1 < 0: all of them)
static int gemm_range(const void* A, long long lda, const void* sa, const void* W, long long ldw, const void* sw, int matrices, void* out, int out_dtype, void* out_scales,
                      int ldo, const void* bias, int bias_dtype, int M, int N, int K, int glu, int act, float limit, const void* row_scale, const void* order,
                      const void* tiles, const void* n_tiles, int max_tiles, int wide, int splits, void* err, void* stream, long long t0, long long t1) {
    MM_REQUIRE(M > 0 && M < FP8_MAX && N > 0 && N < FP8_MAX && K > 0 && K < FP8_MAX && matrices > 0 && lda >= K && ldw >= K && ldo >= N, "gemm_fp8: bad sizes");
    MM_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && (((uintptr_t)A | (uintptr_t)W) & 15) == 0, "gemm_fp8: rows must start on 16-byte boundaries");
    MM_REQUIRE((long long)matrices * N + 256 < 0x7fffffffLL, "gemm_fp8: too many weight rows");
    MM_REQUIRE(out_dtype == MM_F32 || out_dtype == MM_BF16, "gemm_fp8: the result is bf16 or fp32");
    MM_REQUIRE(!glu || (matrices % 2 == 0 && act >= 0 && act <= MM_GLU_GELU_TANH && ldo % 16 == 0 && ((uintptr_t)out & 15) == 0 && out_scales && !bias),
               "gemm_fp8: bad gated product");
    MM_REQUIRE(splits == 1 || splits == 2 || splits == 4 || splits == 8, "gemm_fp8: 1, 2, 4 or 8 splits");
    MM_REQUIRE(tiles == nullptr || (n_tiles && max_tiles > 0 && splits == 1), "gemm_fp8: a grouped product has a list and no splits");
    CUtensorMap ta, tw;
    if (!make_map_bytes(&ta, A, M, K, lda) || !make_map_bytes(&tw, W, (long long)matrices * N, K, ldw)) {
        mm_set_last_error("gemm_fp8: cuTensorMapEncodeTiled failed or is not available");
        return MM_ERR_DRIVER;
    }
    Fp8Args g = {};
    g.out = out;
    g.out_scales = (float*)out_scales;
    g.sa = (const float*)sa;
    g.sw = (const float*)sw;
    g.bias = bias;
    g.row_scale = (const float*)row_scale;
    g.order = (const int32_t*)order;
    g.tiles = (const int32_t*)tiles;
    g.n_tiles = (const int32_t*)n_tiles;
    g.err = (int*)err;
    g.out_kind = out_dtype == MM_F32 ? OUT_F32 : OUT_BF16;
    g.bias_dtype = bias_dtype;
    g.act = act;
    g.limit = limit;
    g.M = M;
    g.N = N;
    g.K = K;
    g.KB = ceil_div(K, FP8_BLOCK);
    g.NB = ceil_div(N, FP8_BLOCK);
    g.ldo = ldo;
    g.S = splits;
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int bn = glu ? 128 : (wide ? 256 : 128);
    const long long total = (long long)(tiles ? max_tiles : ceil_div(M, T_ROWS)) * ceil_div(N, bn);
    MM_REQUIRE(total < 0x40000000LL, "gemm_fp8: too many tiles");
    g.t0 = (int)t0;
    g.t1 = (int)(t1 < 0 ? total : t1);
    cudaStream_t s = (cudaStream_t)stream;
    const int count = g.t1 - g.t0, grid = splits > 1 ? count * splits : (count < sms ? count : sms);
    if (glu) return splits > 1 ? launch<256, true, true>(ta, tw, g, grid, s) : launch<256, true, false>(ta, tw, g, grid, s);
    if (wide) return splits > 1 ? launch<256, false, true>(ta, tw, g, grid, s) : launch<256, false, false>(ta, tw, g, grid, s);
    return splits > 1 ? launch<128, false, true>(ta, tw, g, grid, s) : launch<128, false, false>(ta, tw, g, grid, s);
}

// A e4m3 [M, lda], sa fp32 [M, KB]; W e4m3 [matrices * N, ldw], sw fp32 [matrices, NB, KB] (GLU: pairs of matrices, gate and up).
// glu 0: out [M, ldo] bf16 or fp32 (+ bias [N]); glu 1: out e4m3 [M, ldo] (ldo = N rounded up to 16) and out_scales fp32 [M, NB].
// tiles, n_tiles, max_tiles: the grouped form's row tiles.  wide: 256 columns a tile instead of 128 (GLU: always).  splits: CTAs that share a tile's
// blocks (1, 2, 4 or 8; only without a list).
MM_EXPORT int mm_gemm_fp8_tcgen05(const void* A, long long lda, const void* sa, const void* W, long long ldw, const void* sw, int matrices, void* out,
                                  int out_dtype, void* out_scales, int ldo, const void* bias, int bias_dtype, int M, int N, int K, int glu, int act, float limit,
                                  const void* row_scale, const void* order, const void* tiles, const void* n_tiles, int max_tiles, int wide, int splits,
                                  void* err, void* stream) {
    return gemm_range(A, lda, sa, W, ldw, sw, matrices, out, out_dtype, out_scales, ldo, bias, bias_dtype, M, N, K, glu, act, limit, row_scale, order, tiles, n_tiles,
                      max_tiles, wide, splits, err, stream, 0, -1);
}

namespace {

// How many clusters of S CTAs are resident at once (37 of 4 would be 148 CTAs, but a cluster stays within one part of the chip).
template <int BN, bool GLU>
int resident_clusters(int S) {
    static std::atomic<int> known[9];
    int n = known[S].load(std::memory_order_relaxed);
    if (n > 0) return n;
    typedef Layout<BN> L;
    constexpr size_t smem = (size_t)L::PIPE_BYTES + SUM_WARPS * L::STAGING + 1024 + sizeof(Ctl);
    n = FP8_SM_COUNT / S;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(FP8_SM_COUNT / S * S);
    cfg.blockDim = dim3(T_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int found = 0;
    if (mm_allow_smem<gemm_fp8_tcgen05_kernel<BN, GLU, true>>(smem) &&
        cudaOccupancyMaxActiveClusters(&found, gemm_fp8_tcgen05_kernel<BN, GLU, true>, &cfg) == cudaSuccess && found > 0) n = found;
    else (void)cudaGetLastError();
    known[S].store(n, std::memory_order_relaxed);
    return n;
}

}  // namespace

// The tile's width and the number of CTAs to a tile with the least estimated time: rounds of tiles x (a start and an end + blocks x 0.58 us, of 128 columns 0.4, or
// 0.31 where several row tiles share the weights on their way), as measured with 4 to 100, and 300 to 4,096 rows.  Us estimated and measured: 16 x 3,584 x 18,944 in 128 columns and 4 CTAs 18 and 18, in 2 CTAs 33
// and 28, in 8 (two rounds) 22 and 25; 16 x 18,944 x 3,584 in 256 columns and 2 CTAs 13 and 19 (the weights' way from memory is 10), in 128 columns and one 13 and 22.
// An end is longer than that where a tile's rows of results start at odd places: 333 x 19,001 x 912 is estimated at 13 us and takes 29 (19,008
// columns: 18), whatever the width.
// Beyond whole rounds, what is left may be split: 2,000 x 5,120 x 13,824 (two rounds and 24 tiles) 166 us in one launch, 145 with the 24 over clusters of 4 behind it;
// 1,400 x 3,584 x 3,584 (one round and 6 tiles, or 308 of 128 columns) 37 and 34, narrow 32.
int fp8_gemm(const Fp8In& x, const Fp8Mat& w, const Fp8Out& out, bool glu, int* err, cudaStream_t s) {
    const long long m_tiles = ceil_div(x.rows, T_ROWS), blocks = ceil_div(w.K, FP8_BLOCK);
    const float rows = x.rows < T_ROWS ? (float)x.rows / T_ROWS : 1.0f;       // of a tile: what the CTAs of a cluster hand one another
    int best_wide = 1, best_splits = 1;
    long long best_whole = 0, best_tiles = 0;
    float best = 1e30f;
    for (int wide = glu ? 1 : 0; wide < 2; ++wide) {
        const long long tiles = m_tiles * ceil_div(w.N, glu || !wide ? 128 : 256), rounds = tiles / FP8_SM_COUNT, rest = tiles % FP8_SM_COUNT;
        const float block = wide ? 0.58f : m_tiles > 1 ? 0.31f : 0.4f, whole = 2.0f + (float)blocks * block;
        for (int splits = 1; splits <= 8 && splits <= blocks; splits *= 2) {
            const int fit = splits == 1 ? FP8_SM_COUNT : glu ? resident_clusters<256, true>(splits) : wide ? resident_clusters<256, false>(splits) : resident_clusters<128, false>(splits);
            const float part = splits == 1 ? whole : (wide ? 4.0f + 4.0f * rows : 3.0f + 2.0f * rows) + (float)((blocks + splits - 1) / splits) * block;
            // every tile so, or whole rounds of tiles first and what is left of them split
            for (int tail = 0; tail < (splits > 1 && rounds > 0 && rest > 0 ? 2 : 1); ++tail) {
                const long long here = tail ? rest : tiles;
                const float us = (tail ? (float)rounds * whole + 3.0f : 0.0f) + (float)((here + fit - 1) / fit) * part;
                if (us < best) {
                    best = us;
                    best_wide = wide;
                    best_splits = splits;
                    best_whole = tail ? tiles - rest : 0;
                    best_tiles = tiles;
                }
            }
        }
    }
    auto range = [&](int splits, long long t0, long long t1) {
        return gemm_range(x.data, x.ld, x.scales, w.values, w.ld, w.scales, w.matrices, out.data, out.dtype, out.scales, out.ld, out.bias, out.bias_dtype, x.rows, w.N, w.K, glu,
                          out.act, out.limit, nullptr, nullptr, nullptr, nullptr, 0, best_wide, splits, err, s, t0, t1);
    };
    if (best_whole > 0) {
        const int rc = range(1, 0, best_whole);
        if (rc != MM_OK) return rc;
    }
    return range(best_splits, best_whole, best_tiles);
}
