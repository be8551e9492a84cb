// Products of rows and weights in 8 bits with a scale per row and block of 128 and per weight block of 128 x 128 (fp8.cuh):
//   y[m, n] = sum over blocks b of sa[m, b] sw[n / 128, b] (sum over k in b of qa[m, k] qw[n, k])  (+ bias[n]).
// The inner sums are exact products summed in fp32; each block's sum is scaled and added in fp32.
//
// One thread per result, 16 x 16 of them a CTA, a block of both operands in shared memory at a time.
#include "fp8.cuh"

namespace {

// GLU: W holds two matrices, the gate's and the up projection's, and the result is act(gate, up) in fp32.
// GROUPED: row tile i covers rows tiles[3i] .. tiles[3i + 1] - 1, which meet matrix tiles[3i + 2] (or pair of matrices).
template <bool GLU>
__global__ void __launch_bounds__(256) gemm_fp8_simple_kernel(const uint8_t* __restrict__ A, int lda, const float* __restrict__ sa,
                                                              const uint8_t* __restrict__ W, long long ldw, const float* __restrict__ sw, void* __restrict__ out,
                                                              int out_dtype, int ldo, const void* __restrict__ bias, int bias_dtype, int M, int N, int K,
                                                              const int32_t* __restrict__ tiles, const int32_t* __restrict__ n_tiles, int act, float limit,
                                                              const float* __restrict__ row_scale, const int32_t* __restrict__ order) {
    __shared__ float As[16][FP8_BLOCK + 1], Ws[GLU ? 2 : 1][16][FP8_BLOCK + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int kb = (K + FP8_BLOCK - 1) / FP8_BLOCK, nb = (N + FP8_BLOCK - 1) / FP8_BLOCK, n0 = blockIdx.x * 16;
    int lo = 0, hi = M, e = 0;
    if (tiles != nullptr) {
        if ((int)blockIdx.z >= *n_tiles) return;
        lo = tiles[3 * blockIdx.z];
        hi = tiles[3 * blockIdx.z + 1];
        e = tiles[3 * blockIdx.z + 2];
    }
    const uint8_t* We = W + (size_t)e * (GLU ? 2 : 1) * N * ldw;
    const float* se = sw + (size_t)e * (GLU ? 2 : 1) * nb * kb;
    const int m0 = lo + blockIdx.y * 16;
    if (m0 >= hi) return;
    float total[2] = {0.0f, 0.0f};
    for (int b = 0; b < kb; ++b) {
        for (int i = threadIdx.x; i < 16 * FP8_BLOCK; i += 256) {
            const int r = i >> 7, c = i & 127, k = b * FP8_BLOCK + c;
            As[r][c] = m0 + r < hi && k < K ? fp8_to_f32(A[(size_t)(m0 + r) * lda + k]) : 0.0f;
            for (int j = 0; j < (GLU ? 2 : 1); ++j)
                Ws[j][r][c] = n0 + r < N && k < K ? fp8_to_f32(We[((size_t)j * N + n0 + r) * ldw + k]) : 0.0f;
        }
        __syncthreads();
        const int m = m0 + ty, n = n0 + tx;
        if (m < hi && n < N)
            for (int j = 0; j < (GLU ? 2 : 1); ++j) {
                float part = 0.0f;
                for (int c = 0; c < FP8_BLOCK; ++c) part = fmaf(As[ty][c], Ws[j][tx][c], part);
                total[j] = fmaf(sa[(size_t)m * kb + b] * se[((size_t)j * nb + n / FP8_BLOCK) * kb + b], part, total[j]);
            }
        __syncthreads();
    }
    const int m = m0 + ty, n = n0 + tx;
    if (m >= hi || n >= N) return;
    float v = total[0];
    if (GLU) v = glu_act<false>(v, total[1], act, limit, row_scale ? row_scale[order ? order[m] : m] : 1.0f);
    if (bias != nullptr) v += bias_dtype == MM_F32 ? ((const float*)bias)[n] : __bfloat162float(((const __nv_bfloat16*)bias)[n]);
    if (out_dtype == MM_F32) ((float*)out)[(size_t)m * ldo + n] = v;
    else ((__nv_bfloat16*)out)[(size_t)m * ldo + n] = __float2bfloat16_rn(v);
}

}  // namespace

MM_EXPORT int mm_gemm_fp8_simple(const void* A, int lda, const void* sa, const void* W, long long ldw, const void* sw, void* out, int out_dtype, int ldo,
                                 const void* bias, int bias_dtype, int M, int N, int K, int glu, const void* tiles, const void* n_tiles, int max_tiles,
                                 int act, float limit, const void* row_scale, const void* order, void* stream) {
    MM_REQUIRE(M >= 0 && N > 0 && K > 0 && ldo >= N && lda >= K && ldw >= K, "gemm_fp8: bad sizes");
    if (M == 0) return MM_OK;
    const dim3 grid(ceil_div(N, 16), tiles ? 8 : ceil_div(M, 16), tiles ? max_tiles : 1);
    mm_launch(glu ? gemm_fp8_simple_kernel<true> : gemm_fp8_simple_kernel<false>, grid, dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)A, lda, (const float*)sa,
              (const uint8_t*)W, ldw, (const float*)sw, out, out_dtype, ldo, bias, bias_dtype, M, N, K, (const int32_t*)tiles, (const int32_t*)n_tiles, act, limit,
              (const float*)row_scale, (const int32_t*)order);
    MM_CHECK_LAUNCH();
    return MM_OK;
}
