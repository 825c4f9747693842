// gemm_i8.h -- shared by the kernels of the 8-bit integer product (quant.cu, gemm_i8.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace jst {

struct I8Args {
    int M, N, K;
    const int8_t* A; int64_t lda;  // [M][K] tokens
    const int8_t* B; int64_t ldb;  // [N][K] channels
    const float* a_scale;
    const float* b_scale;
    const float* bias;  // [N] or null
    int relu;
    float* C; int64_t ldc;
};

// The epilogue that every kernel of the product shares, so that they agree in
// every bit: the sum rounded to fp32, the rounded product of the two scales.
__device__ __forceinline__ float i8_finish(int acc, float sa, float sb, bool has_bias, float bias, int relu) {
    float v = __fmul_rn(__int2float_rn(acc), __fmul_rn(sa, sb));
    if (has_bias) v = __fadd_rn(v, bias);
    return relu ? fmaxf(v, 0.0f) : v;
}

// The tensor-core kernels (K > 0, M > 0, N > 0).
int gemm_i8_tc_run(const I8Args& a, cudaStream_t s);

}  // namespace jst
