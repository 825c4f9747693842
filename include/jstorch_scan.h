/*
 * jstorch_scan.h -- a gated linear recurrence over time, exported by
 * jstorch_b200/libjstorch_gemm.so.  It is the state update of the GRU
 * (src/nn.js:485, h' = (1 - z) * n + z * h) with gates that do not read the
 * previous state, so the projections of all steps are one GEMM and the time
 * axis can be scanned in parallel.  The reference has no such operator.
 */
#ifndef JSTORCH_SCAN_H
#define JSTORCH_SCAN_H

#include "jstorch_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* What the second half of a gate row means: n = tanh(c) or n = c. */
enum { JST_SCAN_TANH = 0, JST_SCAN_IDENTITY = 1 };

/*
 * For every sequence b and unit j, over the steps of the sequence in order:
 *   z = sigmoid(a)    n = tanh(c) or c    h_t = z * h_{t-1} + (1 - z) * n
 * z and 1 - z are 0 where they are below 2^-126 (a beyond 87.3 either way): such a
 * gate keeps nothing of the state, whatever its size, or takes nothing of n.
 *   gates    row (t, b) at gates + (t * batch + b) * ld_gates: a in columns
 *            [0, hidden), c in [hidden, 2 * hidden); ld_gates >= 2 * hidden
 *            (every pitch is below 2^24)
 *   h0       [batch][hidden] or NULL (zeros)
 *   lengths  [batch] int32 on the device, or NULL (every sequence has seq
 *            steps).  Sequence b has min(max(lengths[b], 0), seq) steps, the
 *            first ones.  The gates behind them are not read, whatever they
 *            hold; the state passes over them unchanged
 *   reverse  != 0: the steps run from a sequence's last one to its first
 *   out      row (t, b) at out + (t * batch + b) * ld_out: h_t, and 0 behind
 *            the sequence's end; ld_out >= hidden
 *   h_n      [batch][hidden] or NULL: the state after the last step (h0 for a
 *            sequence of no steps).  It may be h0's own memory (a state kept
 *            from call to call); no other outputs may overlap inputs
 * Asynchronous on `stream`; needs no workspace; repeats bit for bit.
 */
int jst_scan_forward(const float* gates, int64_t ld_gates, int seq, int batch, int hidden, const float* h0,
                     const int32_t* lengths, int reverse, int candidate, float* out, int64_t ld_out, float* h_n,
                     jst_stream_t stream);

/*
 * Gradients of jst_scan_forward.  gates, h0, lengths, reverse, candidate and
 * out are those of the forward call (out is read for h_{t-1}).
 *   dout     dL/dout, rows as out's with pitch ld_dout, or NULL (zero); not
 *            read behind a sequence's end
 *   dh_n     [batch][hidden] dL/dh_n, or NULL (zero)
 *   dgates   rows as gates' with pitch ld_dgates: dL/da | dL/dc, 0 behind a
 *            sequence's end
 *   dh0      [batch][hidden] dL/dh0, or NULL; it may be dh_n's own memory
 * Asynchronous on `stream`; needs no workspace; repeats bit for bit.
 */
int jst_scan_backward(const float* gates, int64_t ld_gates, int seq, int batch, int hidden, const float* h0,
                      const int32_t* lengths, int reverse, int candidate, const float* out, int64_t ld_out,
                      const float* dout, int64_t ld_dout, const float* dh_n, float* dgates, int64_t ld_dgates,
                      float* dh0, jst_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* JSTORCH_SCAN_H */
