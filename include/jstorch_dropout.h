/*
 * jstorch_dropout.h -- dropout from a counter-based generator, exported by
 * jstorch_b200/libjstorch_gemm.so.  The mask is a function of (seed, offset,
 * element index), so nothing is stored for the backward pass: the gradient is
 * the same call on the upstream gradient.  The reference has no dropout.
 */
#ifndef JSTORCH_DROPOUT_H
#define JSTORCH_DROPOUT_H

#include "jstorch_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * y[i] = r_i >= T ? x[i] * s : 0    T = floor(p * 2^32), s = 1 / (1 - p) in fp32
 * over the rows x cols elements of a matrix in row-major order, i = row * cols
 * + col whatever the pitches ldx, ldy >= cols are.  r_i is word i % 4 of
 * Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011) with the 128-bit
 * counter (i / 4, offset + *step), low words first, and the 64-bit key seed.
 *   p        0 <= p <= 1; p == 1 writes zeros.  A dropped element is 0
 *            whatever x holds there (infinities and NaN too)
 *   offset   distinguishes calls under one seed: every (seed, offset) pair
 *            has a mask of its own
 *   step     NULL, or a device int64 that is added to offset (modulo 2^64)
 *            when the kernel runs: a captured graph that advances it gets a
 *            new mask at every replay
 *   y        may be x itself (with ldy == ldx), or lie beside x in the same rows;
 *            what shares a byte with x otherwise, or with step, is refused
 * Asynchronous on `stream`; needs no workspace.
 */
int jst_dropout(const float* x, int64_t ldx, float* y, int64_t ldy, int64_t rows, int64_t cols, double p,
                uint64_t seed, uint64_t offset, const int64_t* step, jst_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* JSTORCH_DROPOUT_H */
