// Rows and weights as e4m3 numbers with a scale per block (fp8.cuh has the formula).
#include "fp8.cuh"

namespace {

// One warp per (row, block of 128): four numbers a lane.  Where rows start on whole groups of four the loads and stores are wide ones.
template <typename T>
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const T* __restrict__ x, long long ldx, const int32_t* __restrict__ source,
                                                             uint8_t* __restrict__ q, int ldq, float* __restrict__ scales, long long units, int K,
                                                             int blocks, int wide) {
    const int lane = threadIdx.x & 31;
    for (long long u = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); u < units; u += (long long)gridDim.x * 8) {
        const long long row = u / blocks;
        const int b = (int)(u - row * blocks), k = b * FP8_BLOCK + lane * 4;
        const T* src = x + (source ? source[row] : row) * ldx + k;
        float v[4];
        if (wide && k + 4 <= K) {
            if constexpr (sizeof(T) == 2) {
                const uint2 raw = *reinterpret_cast<const uint2*>(src);
                const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
                const float2 c = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
                v[0] = a.x; v[1] = a.y; v[2] = c.x; v[3] = c.y;
            } else {
                const float4 a = *reinterpret_cast<const float4*>(src);
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = k + i < K ? to_f32<T>(src[i]) : 0.0f;
        }
        const uint32_t mine = max(max(fp8_size_bits(v[0]), fp8_size_bits(v[1])), max(fp8_size_bits(v[2]), fp8_size_bits(v[3])));
        const float s = fp8_scale_of(__reduce_max_sync(0xffffffffu, mine));
        if (lane == 0) scales[u] = s;
        uint8_t* dst = q + row * ldq + k;
        if (k + 4 <= ldq)      // ldq is a multiple of 16: the row's padding gets noughts
            *reinterpret_cast<uint32_t*>(dst) = fp8_pack4(__fdiv_rn(v[0], s), __fdiv_rn(v[1], s), __fdiv_rn(v[2], s), __fdiv_rn(v[3], s));
    }
}

// One CTA per block of 128 x 128: its largest number first, then the quotients (the block comes from L1 the second time).
template <typename T>
__global__ void __launch_bounds__(256) fp8_quant_weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ q, int ldq, float* __restrict__ scales,
                                                               int N, int K) {
    const int nb = (N + FP8_BLOCK - 1) / FP8_BLOCK, kb = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    const size_t matrix = blockIdx.y;
    const int bi = blockIdx.x / kb, bj = blockIdx.x % kb;
    const int n0 = bi * FP8_BLOCK, n1 = min(N, n0 + FP8_BLOCK), k0 = bj * FP8_BLOCK, k1 = min(K, k0 + FP8_BLOCK);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* src = w + matrix * N * (size_t)K;
    __shared__ uint32_t best[8];
    uint32_t mine = 0;
    for (int n = n0 + warp; n < n1; n += 8)
        for (int k = k0 + lane; k < k1; k += 32) mine = max(mine, fp8_size_bits(to_f32<T>(src[(size_t)n * K + k])));
    mine = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) best[warp] = mine;
    __syncthreads();
    mine = best[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mine = max(mine, best[i]);
    const float s = fp8_scale_of(mine);
    if (threadIdx.x == 0) scales[matrix * nb * kb + blockIdx.x] = s;
    const int kq = min(ldq, k0 + FP8_BLOCK);
    for (int n = n0 + warp; n < n1; n += 8)
        for (int k = k0 + lane; k < kq; k += 32)
            q[(matrix * N + n) * (size_t)ldq + k] = k < K ? fp8_one(__fdiv_rn(to_f32<T>(src[(size_t)n * K + k]), s)) : 0;
}

}  // namespace

// x [rows, ldx] (K leading columns) -> q [rows, ldq] e4m3 (ldq = K rounded up to 16, the rest noughts), scales fp32 [rows, K / 128 rounded up].
// source [rows] int32 or null: row r is made from row source[r] of x.
MM_EXPORT int mm_fp8_quant_rows(const void* x, int x_dtype, long long ldx, const void* source, void* q, int ldq, void* scales, int rows, int K, void* stream) {
    MM_REQUIRE(rows >= 0 && K > 0 && ldx >= 0 && ldq >= K && ldq % 16 == 0 && ldq < K + 16, "fp8 rows: bad sizes");
    MM_REQUIRE(((uintptr_t)q & 15) == 0, "fp8 rows: the numbers must start on a 16-byte boundary");
    if (rows == 0) return MM_OK;
    const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    const long long units = (long long)rows * blocks;
    const int grid = (int)((units + 7) / 8 < 148 * 16 ? (units + 7) / 8 : 148 * 16);
    cudaStream_t s = (cudaStream_t)stream;
    const int wide = ldx % 4 == 0 && ((uintptr_t)x & 15) == 0;
    if (x_dtype == MM_BF16)
        mm_launch(fp8_quant_rows_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s, (const __nv_bfloat16*)x, ldx, (const int32_t*)source, (uint8_t*)q, ldq,
                  (float*)scales, units, K, blocks, wide);
    else if (x_dtype == MM_F32)
        mm_launch(fp8_quant_rows_kernel<float>, dim3(grid), dim3(256), 0, s, (const float*)x, ldx, (const int32_t*)source, (uint8_t*)q, ldq, (float*)scales,
                  units, K, blocks, wide);
    else
        MM_REQUIRE(false, "fp8 rows: dtype must be float32 or bfloat16");
    MM_CHECK_LAUNCH();
    return MM_OK;
}

// w [matrices, N, K] -> q [matrices, N, ldq] e4m3, scales fp32 [matrices, N / 128, K / 128] (both rounded up)
MM_EXPORT int mm_fp8_quant_weight(const void* w, int w_dtype, void* q, int ldq, void* scales, int matrices, int N, int K, void* stream) {
    MM_REQUIRE(matrices > 0 && matrices <= 65535 && N > 0 && K > 0 && ldq >= K && ldq % 16 == 0 && ldq < K + 16, "fp8 weight: bad sizes");
    const long long tiles = (long long)((N + FP8_BLOCK - 1) / FP8_BLOCK) * ((K + FP8_BLOCK - 1) / FP8_BLOCK);
    MM_REQUIRE(tiles < 0x7fffffffLL, "fp8 weight: the matrix is too large");
    const dim3 grid((unsigned)tiles, matrices);
    cudaStream_t s = (cudaStream_t)stream;
    if (w_dtype == MM_BF16)
        mm_launch(fp8_quant_weight_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, (const __nv_bfloat16*)w, (uint8_t*)q, ldq, (float*)scales, N, K);
    else if (w_dtype == MM_F32)
        mm_launch(fp8_quant_weight_kernel<float>, grid, dim3(256), 0, s, (const float*)w, (uint8_t*)q, ldq, (float*)scales, N, K);
    else
        MM_REQUIRE(false, "fp8 weight: dtype must be float32 or bfloat16");
    MM_CHECK_LAUNCH();
    return MM_OK;
}
