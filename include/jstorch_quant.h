/*
 * jstorch_quant.h -- 8-bit integer matrix products with one scale a row of
 * each operand, exported by jstorch_b200/libjstorch_gemm.so: the serving form
 * of launch_linear (native/ops/matmul.cu:54).  The reference has none.
 */
#ifndef JSTORCH_QUANT_H
#define JSTORCH_QUANT_H

#include "jstorch_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Quantise rows: scale[r] = max_k |x[r, k]| / 127 rounded to fp32, and q[r, k] =
 * x[r, k] / scale[r] rounded to the nearest integer (ties to even), within
 * [-127, 127].  A row of zeros has scale 0 and q = 0; a row that holds an infinity or a NaN has scale NaN and q = 0, so
 * every product of it is NaN (0 behind a ReLU, as in jst_gemm_ex).
 *   x  row r at x + r * ldx, ldx >= cols;   q  row r at q + r * ldq, ldq >= cols
 * rows and cols are at most 0x7fff0000; the arrays do not overlap.  The bytes of
 * a q row behind `cols` are left as they were.  A pitch that is a multiple of 16
 * (and a 16-byte aligned q) lets jst_gemm_i8 read it in place.
 */
int jst_quantize_rows_i8(const float* x, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq, float* scale,
                         jst_stream_t stream);

/*
 * C[m, n] = epilogue(a_scale[m] * b_scale[n] * sum_k A[m, k] * B[n, k])
 *   A [M][K] int8 (tokens), row pitch lda >= K;  B [N][K] int8 (channels: an
 *   nn.Linear weight), row pitch ldb >= K;  C [M][N] fp32, row pitch ldc >= N.
 *   All int8 values are legal (-128 too).  The sum is exact (32-bit integers;
 *   K <= 131071); it is rounded to fp32 once and multiplied by one scale after the
 *   other, in an order that overflows or underflows only where the result does.
 *   a_scale [M], b_scale [N]; bias [N], required by the bias epilogues.
 *   epilogue: JST_EPI_NONE, JST_EPI_BIAS, JST_EPI_RELU or JST_EPI_BIAS_RELU.
 *   An operand whose address or pitch is not a multiple of 16 bytes is first
 *   copied to an aligned workspace where the tensor cores compute the product.
 * M and N are at most 0x7fff0000; C overlaps no operand.
 * K == 0 writes epilogue(0).  Asynchronous on `stream`; repeats bit for bit.
 */
typedef struct jst_gemm_i8_desc {
    int M, N, K;
    const int8_t* A; int64_t lda;
    const int8_t* B; int64_t ldb;
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    int epilogue;
    float* C; int64_t ldc;
    jst_stream_t stream;
} jst_gemm_i8_desc;

int jst_gemm_i8(const jst_gemm_i8_desc* d);

/*
 * y = epilogue(dequantised(quantised(x) . w^T)): jst_quantize_rows_i8 of x
 * [M][K] (row pitch ldx) and jst_gemm_i8 with w [N][K] (row pitch ldw) and
 * w_scale [N], in one call with the same result.  y [M][N], row pitch ldy.
 */
int jst_linear_i8(const float* x, int64_t ldx, int M, int K, const int8_t* w, int64_t ldw, const float* w_scale,
                  int N, const float* bias, int epilogue, float* y, int64_t ldy, jst_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* JSTORCH_QUANT_H */
