// Entry points that chain the launches of one 8-bit operator (fp8.cuh has the formulas).
//
// Up to 8 rows, and up to 16 of matrices that are not large, go to the weight-streaming kernel, more to tcgen05 tiles.  Rows that come in bf16 or fp32 are quantised by a launch in front, or, where they
// are few numbers (every CTA of the streaming kernel then does it for itself), inside it.
#include "fp8.cuh"
#include "fp8_launch.h"

MM_EXPORT int mm_moe_sort(const void* idx, int n_rows, int E, void* offsets, void* order, int top, int tile_rows, void* tiles, void* n_tiles, void* row_token, void* place,
                          void* stream);
MM_EXPORT int mm_moe_combine(const void* y, int y_dtype, const void* wts, const void* place, void* out, int out_dtype, int n_tokens, int top, int d, void* stream);
MM_EXPORT int mm_fp8_gather_rows(const void* q, const void* scales, const void* source, const void* count, void* out_q, void* out_scales, int rows, int ldq, int blocks,
                                 void* stream);
MM_EXPORT int mm_gemm_fp8_tcgen05(const void* A, long long lda, const void* sa, const void* W, long long ldw, const void* sw, int matrices, void* out, int out_dtype,
                                  void* out_scales, int ldo, const void* bias, int bias_dtype, int M, int N, int K, int glu, int act, float limit, const void* row_scale,
                                  const void* order, const void* tiles, const void* n_tiles, int max_tiles, int wide, int splits, void* err, void* stream);

namespace {

// Numbers up to which the streaming kernel's CTAs quantise the rows, each for itself.  Us inside and with a launch in front: 1 x 4,608 x 3,584 5.7 and 6.1, 4 x 1,024 x 896
// 4.0 and 4.3, a feed-forward of 1 row (896, 4,864) 11.5 and 12.1; 8 x 1,024 x 896 5.1 and 4.5, 2 x 4,608 x 3,584 7.1 and 6.1, 16 x 2,048 x 1,024 7.5 and 4.8.  (One row alone stays a little
// faster inside up to 8,192 numbers, 12.8 and 13.2; at 16,384 it is 53 and 50.)
constexpr int INSIDE_NUMBERS = 4096;

long long row_bytes(int K) { return (long long)(K + 15) / 16 * 16; }
// e4m3 rows and their scales behind them
long long scratch_bytes(int m, int K) { return m * row_bytes(K) + (4LL * m * ceil_div(K, FP8_BLOCK) + 15) / 16 * 16; }

// x as e4m3 rows, in `scratch` if it has to be quantised by a launch; `dependent`: whether that launch was made
int quantised(Fp8In& x, int K, bool glu, unsigned char* scratch, bool& dependent, cudaStream_t s) {
    if (x.dtype == FP8_QUANTISED || ((long long)x.rows * K <= INSIDE_NUMBERS && fp8_gemv_takes(x.rows, K, glu, true))) return MM_OK;
    if (scratch == nullptr) {
        mm_set_last_error("fp8 product: rows of this size need scratch to be quantised in");
        return MM_ERR_BAD_ARG;
    }
    float* scales = (float*)(scratch + x.rows * row_bytes(K));
    const int rc = fp8_quant_rows(x.data, x.dtype, x.ld, x.rows, nullptr, scratch, (int)row_bytes(K), scales, x.rows, K, s);
    x = {scratch, scales, row_bytes(K), FP8_QUANTISED, x.rows};
    dependent = true;
    return rc;
}

// Nine to sixteen rows take a second group of columns through the streaming kernel, and large matrices are then faster over tcgen05 tiles.  Us of the two for 12
// rows: 4,608 x 3,584 8.6 and 10.6, 8,192 x 2,048 9.5 and 9.3, 32,768 x 1,024 13.9 and 11.7, 18,944 x 3,584 19.4 and 18.0, 5,120 x 13,824 25.3 and 21.6 (8 rows: 19.9 and 21.8).
constexpr long long TILED_BYTES = 24 << 20;

int product(const Fp8In& x, const Fp8Mat& w, const Fp8Out& o, bool glu, bool dependent, int* err, cudaStream_t s) {
    const bool tiled = x.dtype == FP8_QUANTISED && x.rows > 8 && (long long)w.matrices * w.N * w.K > TILED_BYTES;
    return !tiled && fp8_gemv_takes(x.rows, w.K, glu, x.dtype != FP8_QUANTISED) ? fp8_gemv(x, w, o, glu, dependent, s) : fp8_gemm(x, w, o, glu, err, s);
}

}  // namespace

// x [m, ldx] bf16 or fp32, or e4m3 with x_scales (dtype 2); W e4m3 [N, ldw], w_scales; bias [N] or null; out [m, N] bf16 or fp32.
// scratch: m * (K rounded up to 16) + 4 m (K / 128 rounded up) bytes, rounded up to 16 (may be null for e4m3
// rows and for up to 16 rows of 4,096 numbers together).
MM_EXPORT int mm_fp8_linear(const void* x, int x_dtype, long long ldx, const void* x_scales, int m, const void* W, long long ldw, const void* w_scales, int N, int K,
                            const void* bias, int bias_dtype, void* out, int out_dtype, void* scratch, void* err, void* stream) {
    MM_REQUIRE(m >= 0 && m < FP8_MAX && N > 0 && N < FP8_MAX && K > 0 && K < FP8_MAX, "fp8 product: bad sizes");
    if (m == 0) return MM_OK;
    cudaStream_t s = (cudaStream_t)stream;
    Fp8In in = {x, (const float*)x_scales, ldx, x_dtype, m};
    bool dependent = false;
    const int rc = quantised(in, K, false, (unsigned char*)scratch, dependent, s);
    if (rc != MM_OK) return rc;
    const Fp8Mat w = {W, (const float*)w_scales, ldw, 1, N, K};
    const Fp8Out o = {out, nullptr, bias, N, out_dtype, bias_dtype, 0, 0.0f};
    return product(in, w, o, false, dependent, (int*)err, s);
}

// The gated feed-forward: w_in e4m3 [2 F, ld_in] (the gate's rows, then the up projection's; scales of each matrix), w_out [D, ld_out]; out bf16 [m, D].
// scratch: as above for K and, behind it, for F.
MM_EXPORT int mm_fp8_glu_mlp(const void* x, int x_dtype, long long ldx, const void* x_scales, int m, const void* w_in, long long ld_in, const void* in_scales, int F,
                             int K, const void* w_out, long long ld_out, const void* out_scales, int D, int act, float limit, void* out, void* scratch, void* err,
                             void* stream) {
    MM_REQUIRE(m >= 0 && m < FP8_MAX && F > 0 && F < FP8_MAX && K > 0 && K < FP8_MAX && D > 0 && D < FP8_MAX && act >= 0 && act <= MM_GLU_GELU_TANH, "fp8 feed-forward: bad sizes or activation");
    if (m == 0) return MM_OK;
    cudaStream_t s = (cudaStream_t)stream;
    Fp8In in = {x, (const float*)x_scales, ldx, x_dtype, m};
    bool dependent = false;
    int rc = quantised(in, K, true, (unsigned char*)scratch, dependent, s);
    if (rc != MM_OK) return rc;
    unsigned char* h = (unsigned char*)scratch + scratch_bytes(m, K);
    float* h_scales = (float*)(h + m * row_bytes(F));
    const Fp8Mat wi = {w_in, (const float*)in_scales, ld_in, 2, F, K}, wo = {w_out, (const float*)out_scales, ld_out, 1, D, F};
    const Fp8Out ho = {h, h_scales, nullptr, (int)row_bytes(F), MM_BF16, MM_F32, act, limit}, o = {out, nullptr, nullptr, D, MM_BF16, MM_F32, 0, 0.0f};
    const Fp8In hidden = {h, h_scales, row_bytes(F), FP8_QUANTISED, m};
    rc = product(in, wi, ho, true, dependent, (int*)err, s);
    return rc != MM_OK ? rc : product(hidden, wo, o, false, true, (int*)err, s);
}

namespace {

constexpr int TILE_ROWS = 128;

// What a prompt's routed experts keep in their scratch, one behind the other
struct ExpertsScratch {
    long long offsets, order, row_token, place, tiles, n_tiles, q, q_scales, sorted, sorted_scales, hidden, hidden_scales, y, bytes;
    ExpertsScratch(long long n, int D, int F, int E, int top) {
        const long long rows = n * top, max_tiles = (rows + TILE_ROWS - 1) / TILE_ROWS + E;
        long long at = 0;
        auto take = [&](long long size) {
            const long long here = at;
            at += (size + 255) / 256 * 256;
            return here;
        };
        offsets = take(4 * (E + 1LL));
        order = take(4 * rows);
        row_token = take(4 * rows);
        place = take(4 * rows);
        tiles = take(12 * max_tiles);
        n_tiles = take(4);
        q = take(n * row_bytes(D));
        q_scales = take(4 * n * ceil_div(D, FP8_BLOCK));
        sorted = take(rows * row_bytes(D));
        sorted_scales = take(4 * rows * ceil_div(D, FP8_BLOCK));
        hidden = take(rows * row_bytes(F));
        hidden_scales = take(4 * rows * ceil_div(F, FP8_BLOCK));
        y = take(4 * rows * D);
        bytes = at;
    }
};

bool experts_fit(long long n, long long D, long long F, int E, long long top) {
    return n >= 0 && D > 0 && D < FP8_MAX && F > 0 && F < FP8_MAX && E > 0 && E <= 4096 && top > 0 && top < FP8_MAX && n * top < FP8_MAX;
}

}  // namespace

// Bytes of scratch that mm_fp8_moe_experts wants (0: sizes that it refuses)
MM_EXPORT long long mm_fp8_moe_experts_scratch(int n, int D, int F, int E, int top) {
    return experts_fit(n, D, F, E, top) ? ExpertsScratch(n, D, F, E, top).bytes : 0;
}

// Routed experts over a prompt: rows sorted by expert, every row quantised once and copied to its experts' places, gate and up with the activation, down
// (fp32, by place), the weighted sum in the order of the choice.  x bf16 or fp32 [n, D]; idx int32, wts fp32 [n, top]; w_in e4m3 [E, 2, F, ld_in], w_out
// [E, D, ld_out]; out bf16 [n, D].  One call and one scratch: six launches take the host 39 us; with an allocation for every list it took 115, more than the kernels of a small layer.
MM_EXPORT int mm_fp8_moe_experts(const void* x, int x_dtype, int n, int D, const void* idx, const void* wts, int top, int E, const void* w_in, long long ld_in,
                                 const void* in_scales, int F, const void* w_out, long long ld_out, const void* out_scales, int act, float limit, int on_input, void* out,
                                 void* scratch, void* err, void* stream) {
    MM_REQUIRE(experts_fit(n, D, F, E, top), "fp8 experts: bad sizes");
    if (n == 0) return MM_OK;
    const ExpertsScratch at(n, D, F, E, top);
    unsigned char* base = (unsigned char*)scratch;
    const int rows = n * top, max_tiles = ceil_div(rows, TILE_ROWS) + E, db = ceil_div(D, FP8_BLOCK);
    int32_t* offsets = (int32_t*)(base + at.offsets);
    int rc = mm_moe_sort(idx, rows, E, offsets, base + at.order, top, TILE_ROWS, base + at.tiles, base + at.n_tiles, base + at.row_token, base + at.place, stream);
    if (rc == MM_OK) rc = fp8_quant_rows(x, x_dtype, D, n, nullptr, base + at.q, (int)row_bytes(D), (float*)(base + at.q_scales), n, D, (cudaStream_t)stream);
    if (rc == MM_OK)
        rc = mm_fp8_gather_rows(base + at.q, base + at.q_scales, base + at.row_token, offsets + E, base + at.sorted, base + at.sorted_scales, rows, (int)row_bytes(D), db, stream);
    if (rc == MM_OK)
        rc = mm_gemm_fp8_tcgen05(base + at.sorted, row_bytes(D), base + at.sorted_scales, w_in, ld_in, in_scales, 2 * E, base + at.hidden, MM_BF16, base + at.hidden_scales,
                                 (int)row_bytes(F), nullptr, MM_F32, rows, F, D, 1, act, limit, on_input ? wts : nullptr, base + at.order, base + at.tiles, base + at.n_tiles,
                                 max_tiles, 1, 1, err, stream);
    if (rc == MM_OK)
        rc = mm_gemm_fp8_tcgen05(base + at.hidden, row_bytes(F), base + at.hidden_scales, w_out, ld_out, out_scales, E, base + at.y, MM_F32, nullptr, D, nullptr, MM_F32, rows, D, F,
                                 0, 0, 0.0f, nullptr, base + at.order, base + at.tiles, base + at.n_tiles, max_tiles, 1, 1, err, stream);
    if (rc == MM_OK) rc = mm_moe_combine(base + at.y, MM_F32, on_input ? nullptr : wts, base + at.place, out, MM_BF16, n, top, D, stream);
    return rc;
}
