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

// q = x / s to the nearest integer, ties to even, where s = max|x| * (1 / 127) > 0.
// x * (1 / s) is within a few 2^-24 of the quotient, so only a value within
// 2^-12 of a half can round to another integer than the quotient does; those
// (one in two thousand) divide in 64 bits, which separates every quotient of
// two fp32 numbers from a half that it does not equal.
__device__ __forceinline__ int quantize(float x, float s, float inv) {
    const float t = x * inv;
    float q = rintf(t);
    if (!(fabsf(fabsf(t - q) - 0.5f) > 0.000244140625f)) q = (float)rint((double)x / (double)s);
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// Largest |x| of a row as its bits: the order of non-negative floats is the
// order of their bits, and a NaN's are above infinity's, so one integer
// maximum finds the peak and tells a row that is not finite.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t peak) {
    return peak < 0x7f800000u ? __fmul_rn(__uint_as_float(peak), 1.0f / 127.0f) : __uint_as_float(0x7fffffffu);
}
// 1 / s, or 0 where the row quantises to zeros (s is 0 or NaN).
__device__ __forceinline__ float row_inverse(float s) { return s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f; }

__device__ __forceinline__ int quantize_in(float x, float s, float inv) { return inv > 0.0f ? quantize(x, s, inv) : 0; }

// The tensor-core kernels (K > 0, M > 0, N > 0).
int gemm_i8_tc_run(const I8Args& a, cudaStream_t s);
// The same with the tokens in fp32 (row pitch ldx), quantised by the product's
// own blocks: a.A and a.a_scale are unused.  For calls that this takes.
bool gemm_i8_tc_takes_fp32(const I8Args& a);
int gemm_i8_tc_run_fp32(const I8Args& a, const float* x, int64_t ldx, cudaStream_t s);

}  // namespace jst
