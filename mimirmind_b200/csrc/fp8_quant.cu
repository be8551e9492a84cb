// Rows and weights as e4m3 numbers with a scale per block (fp8.cuh has the formula).
#include "fp8.cuh"
#include "fp8_launch.h"

namespace {

// Two blocks of a row per warp (a unit), eight numbers a lane; where rows start on 16-byte boundaries the loads are wide ones.  Many short warps hide the
// loads: three units a warp, their loads together on their way, were no faster.
// Bound by memory (3 bytes a number) and by the instructions a number (quotient, largest, conversion): 4,096 rows of 3,584 bf16 (44 MB, floor 6.7 us) 12.1 to 12.4 us (3.6 TB/s), with a division a
// number 19.7.
template <typename T>
__global__ void __launch_bounds__(256) fp8_quant_rows_kernel(const T* __restrict__ x, long long ldx, int x_rows, const int32_t* __restrict__ source,
                                                             uint8_t* __restrict__ q, int ldq, float* __restrict__ scales, uint32_t units, int K,
                                                             uint32_t pairs, int blocks, int wide) {
    const int lane = threadIdx.x & 31;
    pdl_trigger();        // a product launched behind this may fetch its first weights meanwhile
    const uint32_t u = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (u >= units) return;
    const uint32_t row = u / pairs;
    const int b = (int)(u - row * pairs) * 2 + (lane >> 4), k = b * FP8_BLOCK + (lane & 15) * 8;
    const int from = source ? source[row] : (int)row, end = (unsigned)from < (unsigned)x_rows ? K : 0;      // (a number that is no row's, as of padding: noughts)
    const T* src = x + from * ldx + k;
    float v[8];
    if (wide && k + 8 <= end) {
        fp8_load8<T>(src, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < end ? to_f32<T>(src[i]) : 0.0f;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, fp8_size_bits(v[i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const float s = fp8_scale_of(largest);
    if ((lane & 15) == 0 && b < blocks) scales[(size_t)row * blocks + b] = s;
    fp8_quotients<8>(v, s);
    if (k + 8 <= ldq)      // ldq is a multiple of 16: the row's padding gets noughts
        *reinterpret_cast<uint2*>(q + (size_t)row * ldq + k) = make_uint2(fp8_pack4(v[0], v[1], v[2], v[3]), fp8_pack4(v[4], v[5], v[6], v[7]));
}

// Quantised rows copied to other places: out row r is row source[r], numbers and scales, for the first *count rows.  A warp per row, 16 bytes a lane.
__global__ void __launch_bounds__(256) fp8_gather_rows_kernel(const uint4* __restrict__ q, const float* __restrict__ s, const int32_t* __restrict__ source, const int32_t* __restrict__ count,
                                                              uint4* __restrict__ oq, float* __restrict__ os, int rows, int pieces, int blocks) {
    const int lane = threadIdx.x & 31, row = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows || row >= *count) return;
    const size_t from = source[row];
#pragma unroll 4
    for (int i = lane; i < pieces; i += 32) oq[(size_t)row * pieces + i] = q[from * pieces + i];
    for (int i = lane; i < blocks; i += 32) os[(size_t)row * blocks + i] = s[from * blocks + i];
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

int fp8_quant_rows(const void* x, int x_dtype, long long ldx, int x_rows, const int32_t* source, void* q, int ldq, float* scales, int rows, int K, cudaStream_t s) {
    MM_REQUIRE(rows >= 0 && rows < FP8_MAX && K > 0 && K < FP8_MAX && ldx >= 0 && ldq >= K && ldq % 16 == 0 && ldq < K + 16, "fp8 rows: bad sizes");
    MM_REQUIRE(((uintptr_t)q & 15) == 0, "fp8 rows: the numbers must start on a 16-byte boundary");
    if (rows == 0) return MM_OK;
    const int blocks = (K + FP8_BLOCK - 1) / FP8_BLOCK;
    const int pairs = (blocks + 1) / 2;
    const long long units = (long long)rows * pairs;
    MM_REQUIRE(units < 0x7fffffffLL, "fp8 rows: too many rows");
    const int grid = (int)((units + 7) / 8);
    const int wide = ldx % (x_dtype == MM_BF16 ? 8 : 4) == 0 && ((uintptr_t)x & 15) == 0;
    if (x_dtype == MM_BF16)
        mm_launch(fp8_quant_rows_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s, (const __nv_bfloat16*)x, ldx, x_rows, source, (uint8_t*)q, ldq,
                  scales, (uint32_t)units, K, (uint32_t)pairs, blocks, wide);
    else if (x_dtype == MM_F32)
        mm_launch(fp8_quant_rows_kernel<float>, dim3(grid), dim3(256), 0, s, (const float*)x, ldx, x_rows, source, (uint8_t*)q, ldq, scales,
                  (uint32_t)units, K, (uint32_t)pairs, blocks, wide);
    else
        MM_REQUIRE(false, "fp8 rows: dtype must be float32 or bfloat16");
    MM_CHECK_LAUNCH();
    return MM_OK;
}

// x [rows, ldx] (K leading columns) -> q [rows, ldq] e4m3 (ldq = K rounded up to 16, the rest noughts), scales fp32 [rows, K / 128 rounded up]; `source` null.
MM_EXPORT int mm_fp8_quant_rows(const void* x, int x_dtype, long long ldx, const void* source, void* q, int ldq, void* scales, int rows, int K, void* stream) {
    MM_REQUIRE(source == nullptr, "fp8 rows: rows made from others want x's number of rows (mm_fp8_quant_rows_from)");
    return fp8_quant_rows(x, x_dtype, ldx, rows, nullptr, q, ldq, (float*)scales, rows, K, (cudaStream_t)stream);
}

// The same with source [rows] int32: row r is made from row source[r] of x's x_rows rows, or of noughts where there is no such row.
MM_EXPORT int mm_fp8_quant_rows_from(const void* x, int x_dtype, long long ldx, int x_rows, const void* source, void* q, int ldq, void* scales, int rows, int K,
                                     void* stream) {
    MM_REQUIRE(source != nullptr && x_rows >= 0, "fp8 rows: bad source");
    return fp8_quant_rows(x, x_dtype, ldx, x_rows, (const int32_t*)source, q, ldq, (float*)scales, rows, K, (cudaStream_t)stream);
}

// q [., ldq] e4m3 (ldq a multiple of 16) with scales fp32 [., blocks]: row r of the result is row source[r], for the first *count of `rows` rows
MM_EXPORT int mm_fp8_gather_rows(const void* q, const void* scales, const void* source, const void* count, void* out_q, void* out_scales, int rows, int ldq, int blocks, void* stream) {
    MM_REQUIRE(rows >= 0 && ldq > 0 && ldq % 16 == 0 && blocks > 0 && (((uintptr_t)q | (uintptr_t)out_q) & 15) == 0, "fp8 rows: bad sizes");
    if (rows == 0) return MM_OK;
    mm_launch(fp8_gather_rows_kernel, dim3(ceil_div(rows, 8)), dim3(256), 0, (cudaStream_t)stream, (const uint4*)q, (const float*)scales, (const int32_t*)source,
              (const int32_t*)count, (uint4*)out_q, (float*)out_scales, rows, ldq / 16, blocks);
    MM_CHECK_LAUNCH();
    return MM_OK;
}

// w [matrices, N, K] -> q [matrices, N, ldq] e4m3, scales fp32 [matrices, N / 128, K / 128] (both rounded up)
MM_EXPORT int mm_fp8_quant_weight(const void* w, int w_dtype, void* q, int ldq, void* scales, int matrices, int N, int K, void* stream) {
    MM_REQUIRE(matrices > 0 && matrices <= 65535 && N > 0 && N < FP8_MAX && K > 0 && K < FP8_MAX && ldq >= K && ldq % 16 == 0 && ldq < K + 16, "fp8 weight: bad sizes");
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
