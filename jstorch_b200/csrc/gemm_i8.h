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
// every bit: the sum rounded to fp32, times the token's scale, times the
// channel's; or times the channel's first where |acc sa|, |acc| <= 2^31, could
// overflow.  (A whole number times a scale loses nothing to underflow, where the
// product of two scales may: what meets the type's range is the result alone.)
// One of the three factors is 1.
__device__ __forceinline__ float i8_finish(int acc, float sa, float sb, bool has_bias, float bias, int relu) {
    const bool late = fabsf(sa) > 7.9228162514264338e28f;  // 2^96
    float v = __fmul_rn(__int2float_rn(acc), late ? 1.0f : sa);
    v = __fmul_rn(__fmul_rn(v, sb), late ? sa : 1.0f);
    if (has_bias) v = __fadd_rn(v, bias);
    return relu ? fmaxf(v, 0.0f) : v;
}

// Largest |x| of a row as its bits: the order of non-negative floats is the
// order of their bits, and a NaN's are above infinity's, so one integer
// maximum finds the peak and tells a row that is not finite.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t peak) {
    return peak < 0x7f800000u ? __fdiv_rn(__uint_as_float(peak), 127.0f) : __uint_as_float(0x7fffffffu);
}
// 1 / s, or 0 where the row quantises to zeros (s is 0 or NaN).
__device__ __forceinline__ float row_inverse(float s) { return s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f; }

// q = x / s to the nearest integer, ties to even, within [-127, 127], where s =
// max|x| / 127 > 0, by a division in 64 bits.  (A call: it is rare.)
static __device__ __noinline__ uint32_t quantize_exactly(float x, float s) {
    return (uint32_t)(uint8_t)(int8_t)fmin(fmax(rint((double)x / (double)s), -127.0), 127.0);
}

// Four values of a row as the bytes of a word, each the nearest integer to x / s.
// t = x * (1 / s) is within a few 2^-24 of the quotient.  Adding 1.5 * 2^23
// rounds it to an integer n and leaves n's low byte in the low byte of the sum
// (no conversion, of which an SM does a quarter as many).  Only where t is within
// 2^-12 of a half h (one value in two thousand) can the quotient be on the other
// side of h than t: there the sign of x - h s decides, which one fused
// multiply-add has exactly, and equality goes to the even side.  That sign could
// underflow for a tiny s, whose rows divide.
__device__ __forceinline__ uint32_t quantize4(const float4& x, float s, float inv) {
    if (!(inv > 0.0f)) return 0u;
    constexpr float shift = 12582912.0f, close = 0.000244140625f;
    const float v[4] = {x.x, x.y, x.z, x.w};
    uint32_t b[4];
    if (s >= 7.8886090522101181e-31f) {  // 2^-100
        float n[4], d[4], nearest = 1.0f;  // to a half
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = __fmul_rn(v[i], inv), r = __fadd_rn(t, shift);
            b[i] = __float_as_uint(r);
            n[i] = __fadd_rn(r, -shift);
            d[i] = __fadd_rn(t, -n[i]);
            nearest = fminf(nearest, 0.5f - fabsf(d[i]));
        }
        if (nearest <= close)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float side = d[i] > 0.0f ? 1.0f : -1.0f;
                const float past = side * fmaf(-(n[i] + 0.5f * side), s, v[i]);
                const bool move = past > 0.0f || (past == 0.0f && (b[i] & 1u));
                if (0.5f - fabsf(d[i]) <= close && move) b[i] += d[i] > 0.0f ? 1u : ~0u;
            }
    } else {
        for (int i = 0; i < 4; ++i) b[i] = quantize_exactly(v[i], s);
    }
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
}

// The tensor-core kernels (K > 0, M > 0, N > 0).
int gemm_i8_tc_run(const I8Args& a, cudaStream_t s);
// Whether gemm_i8_tc_run reads A and B where they are.
bool gemm_i8_tc_in_place(const I8Args& a);
// The same with the tokens in fp32 (row pitch ldx), quantised by the product's
// own blocks: a.A and a.a_scale are unused.  For calls that this takes.
bool gemm_i8_tc_takes_fp32(const I8Args& a);
int gemm_i8_tc_run_fp32(const I8Args& a, const float* x, int64_t ldx, cudaStream_t s);

}  // namespace jst
