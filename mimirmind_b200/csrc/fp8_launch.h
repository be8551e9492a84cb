// The 8-bit products' launches, as the entry points that chain them see them (host only).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

constexpr int FP8_QUANTISED = 2;          // dtype of rows that are e4m3 already
constexpr int FP8_SM_COUNT = 148;

struct Fp8In {                            // rows: bf16 or fp32, or e4m3 with scales fp32 [rows, K / 128 rounded up]
    const void* data;
    const float* scales;
    long long ld;
    int dtype, rows;
};
struct Fp8Mat {                           // e4m3 [matrices * N, ld], scales fp32 [matrices, N / 128, K / 128]
    const void* values;
    const float* scales;
    long long ld;
    int matrices, N, K;
};
struct Fp8Out {                           // rows [., ld] bf16 or fp32; gated products: e4m3 [., ld] and scales
    void* data;
    float* scales;
    const void* bias;
    int ld, dtype, bias_dtype, act;
    float limit;
};

int fp8_quant_rows(const void* x, int x_dtype, long long ldx, int x_rows, const int32_t* source, void* q, int ldq, float* scales, int rows, int K, cudaStream_t s);
// up to 16 rows; `dependent`: launched behind a kernel of this library in the same stream, whose end it waits for itself.  Rows that are not quantised
// yet are quantised in the kernel (few numbers: it has them in shared memory).
int fp8_gemv(const Fp8In& x, const Fp8Mat& w, const Fp8Out& out, bool glu, bool dependent, cudaStream_t s);
bool fp8_gemv_takes(int rows, int K, bool glu, bool quant);      // rows short enough for its shared memory
// any number of rows, quantised
int fp8_gemm(const Fp8In& x, const Fp8Mat& w, const Fp8Out& out, bool glu, int* err, cudaStream_t s);
