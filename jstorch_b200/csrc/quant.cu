// quant.cu -- the entry points of include/jstorch_quant.h: row quantisation
// and the 8-bit integer matrix product with a scale per row of each operand.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "../../include/jstorch_quant.h"
#include "gemm_internal.h"

namespace jst {
namespace {

// q = x / s to the nearest integer, ties to even, where s = max|x| / 127 > 0.
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

constexpr int kQuantThreads = 256;

__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const float* __restrict__ x, int64_t ldx,
                                                                      int cols, int8_t* __restrict__ q, int64_t ldq,
                                                                      float* __restrict__ scale) {
    __shared__ uint32_t part[kQuantThreads / 32];
    const float* row = x + (int64_t)blockIdx.x * ldx;
    int8_t* out = q + (int64_t)blockIdx.x * ldq;
    uint32_t m = 0;
    for (int k = threadIdx.x; k < cols; k += kQuantThreads) m = max(m, abs_bits(row[k]));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kQuantThreads / 32; ++w) m = max(m, part[w]);
    const bool finite = m < 0x7f800000u;
    const float s = finite ? __fdiv_rn(__uint_as_float(m), 127.0f) : __uint_as_float(0x7fffffffu);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    const bool zero = !finite || s == 0.0f;
    const float inv = zero ? 0.0f : __fdiv_rn(1.0f, s);
    for (int k = threadIdx.x; k < cols; k += kQuantThreads) out[k] = zero ? (int8_t)0 : (int8_t)quantize(row[k], s, inv);
}

struct I8Args {
    int M, N, K;
    const int8_t* A; int64_t lda;
    const int8_t* B; int64_t ldb;
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    int relu;
    float* C; int64_t ldc;
};

__device__ __forceinline__ float finish(int acc, float sa, float sb, bool has_bias, float bias, int relu) {
    float v = __fmul_rn(__int2float_rn(acc), __fmul_rn(sa, sb));
    if (has_bias) v = __fadd_rn(v, bias);
    return relu ? fmaxf(v, 0.0f) : v;
}

// Any sizes, any addresses: a block of 256 threads computes 64 x 64 outputs
// from 64-byte k-slabs in shared memory, 4 x 4 outputs a thread with dp4a.
__global__ void __launch_bounds__(256) gemm_i8_simt_kernel(const I8Args p) {
    constexpr int T = 64, BK = 64, LD = BK / 4 + 1;
    __shared__ int as[T][LD], bs[T][LD];
    const int m0 = blockIdx.y * T, n0 = blockIdx.x * T;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += BK) {
        for (int i = threadIdx.x; i < T * BK / 4; i += 256) {
            const int r = i / (BK / 4), w = i % (BK / 4), k = k0 + 4 * w;
            uint32_t va = 0, vb = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (k + j >= p.K) continue;
                if (m0 + r < p.M) va |= (uint32_t)(uint8_t)p.A[(int64_t)(m0 + r) * p.lda + k + j] << (8 * j);
                if (n0 + r < p.N) vb |= (uint32_t)(uint8_t)p.B[(int64_t)(n0 + r) * p.ldb + k + j] << (8 * j);
            }
            as[r][w] = (int)va;
            bs[r][w] = (int)vb;
        }
        __syncthreads();
#pragma unroll 4
        for (int w = 0; w < BK / 4; ++w) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = as[ty * 4 + i][w];
                b[i] = bs[tx + 16 * i][w];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty * 4 + i;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx + 16 * j;
            if (n < p.N)
                p.C[(int64_t)m * p.ldc + n] =
                    finish(acc[i][j], p.a_scale[m], p.b_scale[n], p.bias != nullptr, p.bias ? p.bias[n] : 0.0f, p.relu);
        }
    }
}

int launched(const char* what) {
    return cudaPeekAtLastError() == cudaSuccess ? set_status(JST_OK, nullptr) : set_status(JST_ERR_CUDA, what);
}

int check_quantize(const float* x, int64_t ldx, int rows, int cols, const int8_t* q, int64_t ldq, const float* scale) {
    if (rows < 0 || cols < 0) return set_status(JST_ERR_ARG, "quantize_rows: negative size");
    if (rows == 0) return JST_OK;
    if (!scale || (cols > 0 && (!x || !q))) return set_status(JST_ERR_ARG, "quantize_rows: null pointer");
    if (rows > 1 && (ldx < cols || ldq < cols)) return set_status(JST_ERR_ARG, "quantize_rows: pitch < cols");
    if (rows > 1 && (ldx > INT64_MAX / 8 / rows || ldq > INT64_MAX / 8 / rows))
        return set_status(JST_ERR_ARG, "quantize_rows: size exceeds 64 bits");
    return JST_OK;
}

int run_quantize(const float* x, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq, float* scale, cudaStream_t s) {
    if (rows == 0) return set_status(JST_OK, nullptr);
    {
        ProfScope prof(s, KID_QUANT);
        quantize_rows_kernel<<<(unsigned)rows, kQuantThreads, 0, s>>>(x, ldx, cols, q, ldq, scale);
    }
    return launched("quantize_rows launch failed");
}

// The parts of a descriptor that jst_gemm_i8 and jst_linear_i8 share.
int check_product(int M, int N, int K, int64_t ldb, const void* B, const float* b_scale, const float* bias,
                  int epilogue, const float* C, int64_t ldc) {
    if (M < 0 || N < 0 || K < 0) return set_status(JST_ERR_ARG, "gemm_i8: negative size");
    if (K > 131071) return set_status(JST_ERR_ARG, "gemm_i8: K > 131071 (the sum could exceed 32 bits)");
    if (epilogue < JST_EPI_NONE || epilogue > JST_EPI_BIAS_RELU) return set_status(JST_ERR_ARG, "gemm_i8: unknown epilogue");
    if ((epilogue & JST_EPI_BIAS) && !bias) return set_status(JST_ERR_ARG, "gemm_i8: bias epilogue without a bias pointer");
    if (M == 0 || N == 0) return JST_OK;
    if (!C || !b_scale || (K > 0 && !B)) return set_status(JST_ERR_ARG, "gemm_i8: null pointer");
    if ((M > 1 && ldc < N) || (N > 1 && K > 0 && ldb < K)) return set_status(JST_ERR_ARG, "gemm_i8: pitch too small");
    if ((M > 1 && ldc > INT64_MAX / 8 / M) || (N > 1 && ldb > INT64_MAX / 8 / N))
        return set_status(JST_ERR_ARG, "gemm_i8: size exceeds 64 bits");
    return JST_OK;
}

int run_gemm_i8(const I8Args& p, cudaStream_t s) {
    {
        ProfScope prof(s, KID_GEMM_I8);
        gemm_i8_simt_kernel<<<dim3((p.N + 63) / 64, (p.M + 63) / 64), 256, 0, s>>>(p);
    }
    return launched("gemm_i8 launch failed");
}

}  // namespace
}  // namespace jst

extern "C" int jst_quantize_rows_i8(const float* x, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq,
                                    float* scale, jst_stream_t stream) {
    using namespace jst;
    int rc = check_quantize(x, ldx, rows, cols, q, ldq, scale);
    if (rc) return rc;
    rc = require_device();
    if (rc) return rc;
    return run_quantize(x, ldx, rows, cols, q, ldq, scale, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int jst_gemm_i8(const jst_gemm_i8_desc* d) {
    using namespace jst;
    if (!d) return set_status(JST_ERR_ARG, "null descriptor");
    int rc = check_product(d->M, d->N, d->K, d->ldb, d->B, d->b_scale, d->bias, d->epilogue, d->C, d->ldc);
    if (rc) return rc;
    if (d->M > 0 && d->N > 0) {
        if (!d->a_scale || (d->K > 0 && !d->A)) return set_status(JST_ERR_ARG, "gemm_i8: null pointer");
        if (d->M > 1 && d->K > 0 && d->lda < d->K) return set_status(JST_ERR_ARG, "gemm_i8: pitch too small");
        if (d->M > 1 && d->lda > INT64_MAX / 8 / d->M) return set_status(JST_ERR_ARG, "gemm_i8: size exceeds 64 bits");
    }
    rc = require_device();
    if (rc) return rc;
    if (d->M == 0 || d->N == 0) return set_status(JST_OK, nullptr);
    I8Args p{d->M, d->N, d->K, d->A, d->lda, d->B, d->ldb, d->a_scale, d->b_scale,
             (d->epilogue & JST_EPI_BIAS) ? d->bias : nullptr, (d->epilogue & JST_EPI_RELU) ? 1 : 0, d->C, d->ldc};
    return run_gemm_i8(p, reinterpret_cast<cudaStream_t>(d->stream));
}

extern "C" int jst_linear_i8(const float* x, int64_t ldx, int M, int K, const int8_t* w, int64_t ldw,
                             const float* w_scale, int N, const float* bias, int epilogue, float* y, int64_t ldy,
                             jst_stream_t stream) {
    using namespace jst;
    int rc = check_product(M, N, K, ldw, w, w_scale, bias, epilogue, y, ldy);
    if (rc) return rc;
    if (M > 0 && N > 0) {
        if (K > 0 && !x) return set_status(JST_ERR_ARG, "linear_i8: null pointer");
        if (M > 1 && ldx < K) return set_status(JST_ERR_ARG, "linear_i8: pitch too small");
        if (M > 1 && ldx > INT64_MAX / 8 / M) return set_status(JST_ERR_ARG, "linear_i8: size exceeds 64 bits");
    }
    rc = require_device();
    if (rc) return rc;
    if (M == 0 || N == 0) return set_status(JST_OK, nullptr);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t ldq = ((int64_t)K + 15) / 16 * 16;
    const size_t scale_bytes = ((size_t)M * 4 + 255) & ~size_t(255);
    void* ws = nullptr;
    rc = workspace_alloc(scale_bytes + (size_t)M * ldq, s, &ws);
    if (rc) return rc;
    float* scale = static_cast<float*>(ws);
    int8_t* q = static_cast<int8_t*>(ws) + scale_bytes;
    rc = run_quantize(x, ldx, M, K, q, ldq, scale, s);
    if (!rc) {
        I8Args p{M, N, K, q, ldq, w, ldw, scale, w_scale, (epilogue & JST_EPI_BIAS) ? bias : nullptr,
                 (epilogue & JST_EPI_RELU) ? 1 : 0, y, ldy};
        rc = run_gemm_i8(p, s);
    }
    const int frc = workspace_free(ws, s);
    return rc ? rc : frc ? frc : set_status(JST_OK, nullptr);
}
