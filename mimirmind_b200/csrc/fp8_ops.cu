// Entry points that chain the launches of one 8-bit operator (fp8.cuh has the formulas).
//
// Up to 16 rows go to the weight-streaming kernel, more to tcgen05 tiles.  Rows that come in bf16 or fp32 are quantised by a launch in front, or, where they
// are few numbers (every CTA of the streaming kernel then does it for itself), inside it.
#include "fp8.cuh"
#include "fp8_launch.h"

namespace {

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
    const int rc = fp8_quant_rows(x.data, x.dtype, x.ld, nullptr, scratch, (int)row_bytes(K), scales, x.rows, K, s);
    x = {scratch, scales, row_bytes(K), FP8_QUANTISED, x.rows};
    dependent = true;
    return rc;
}

int product(const Fp8In& x, const Fp8Mat& w, const Fp8Out& o, bool glu, bool dependent, int* err, cudaStream_t s) {
    return fp8_gemv_takes(x.rows, w.K, glu, x.dtype != FP8_QUANTISED) ? fp8_gemv(x, w, o, glu, dependent, s) : fp8_gemm(x, w, o, glu, err, s);
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
