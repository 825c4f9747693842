// quant.cu -- the entry points of include/jstorch_quant.h: row quantisation
// and the 8-bit integer matrix product with a scale per row of each operand.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "../../include/jstorch_quant.h"
#include "gemm_i8.h"
#include "gemm_internal.h"
#include "ptx.cuh"

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

__device__ __forceinline__ float row_scale(uint32_t peak) {
    return peak < 0x7f800000u ? __fdiv_rn(__uint_as_float(peak), 127.0f) : __uint_as_float(0x7fffffffu);
}
// 1 / s, or 0 where the row quantises to zeros (s is 0 or NaN).
__device__ __forceinline__ float row_inverse(float s) { return s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f; }

__device__ __forceinline__ int quantize_in(float x, float s, float inv) { return inv > 0.0f ? quantize(x, s, inv) : 0; }

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
    const float s = row_scale(m), inv = row_inverse(s);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    for (int k = threadIdx.x; k < cols; k += kQuantThreads) out[k] = (int8_t)quantize_in(row[k], s, inv);
}

// ------------------------------------------------------------ a few tokens
// C[m, n] for MT <= 8 tokens.  A warp takes kChannels rows of the weight and
// walks along K, 16 bytes a lane and row: one 16-byte piece of a token from
// shared memory meets kChannels pieces of the weight, 4 dp4a each.  The
// lanes' sums meet in one integer reduction, exact in any order.
// Bound by the weight's bytes; each is read once.
// The tokens are held in shared memory kSegment values of K at a time.  FUSED:
// they come as fp32 rows and every block quantises them itself.
// ALIGN: 16 when the weight's rows are 16-byte aligned.  Otherwise 1: a lane
// reads the aligned 4-byte words that hold its 16 bytes and shifts; a word that
// holds a byte of the row does not leave the memory block that the row is in.
constexpr int kFewThreads = 256;
constexpr int kChannels = 4;
constexpr int kSegment = 8192;

struct FewArgs {
    I8Args p;        // FUSED: A and a_scale are unused
    const float* x;  // FUSED: [M][K] fp32
    int64_t ldx;
};

template <int ALIGN>
__device__ __forceinline__ int4 load16(const int8_t* w) {
    if (ALIGN == 16) return __ldg(reinterpret_cast<const int4*>(w));
    const uintptr_t at = reinterpret_cast<uintptr_t>(w);
    const uint32_t* word = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
    const uint32_t shift = (uint32_t)(at & 3) * 8;
    uint32_t v[5];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __ldg(word + i);
    v[4] = shift ? __ldg(word + 4) : 0u;
    return make_int4((int)__funnelshift_r(v[0], v[1], shift), (int)__funnelshift_r(v[1], v[2], shift),
                     (int)__funnelshift_r(v[2], v[3], shift), (int)__funnelshift_r(v[3], v[4], shift));
}

__device__ __forceinline__ int dot16(int4 a, int4 b, int c) {
    return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, c))));
}

template <int MT, int ALIGN, bool FUSED>
__global__ void __launch_bounds__(kFewThreads) gemm_i8_few_kernel(const FewArgs f) {
    extern __shared__ __align__(16) int8_t tokens[];  // [MT][seg], seg a multiple of 16
    __shared__ uint32_t part[MT][kFewThreads / 32];
    __shared__ float scales[MT], inverses[MT];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const I8Args& p = f.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = (blockIdx.x * (kFewThreads / 32) + warp) * kChannels;
    if (FUSED) {
        for (int m = 0; m < MT; ++m) {
            uint32_t peak = 0;
            if (m < p.M)
                for (int k = threadIdx.x; k < p.K; k += kFewThreads) peak = max(peak, abs_bits(__ldg(f.x + m * f.ldx + k)));
            peak = __reduce_max_sync(0xffffffffu, peak);
            if (lane == 0) part[m][warp] = peak;
        }
        __syncthreads();
        if (threadIdx.x < MT) {
            uint32_t peak = 0;
            for (int w = 0; w < kFewThreads / 32; ++w) peak = max(peak, part[threadIdx.x][w]);
            scales[threadIdx.x] = row_scale(peak);
            inverses[threadIdx.x] = row_inverse(scales[threadIdx.x]);
        }
        __syncthreads();
    }
    int acc[kChannels][MT] = {};
    for (int k0 = 0; k0 < p.K; k0 += kSegment) {
        const int len = min(kSegment, p.K - k0), seg = (len + 15) & ~15;
        for (int i = threadIdx.x * 4; i < MT * seg; i += kFewThreads * 4) {  // seg is a multiple of 4
            const int m = i / seg, k = i - m * seg;
            uint32_t v = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (m < p.M && k + j < len) {
                    const int q = FUSED ? quantize_in(__ldg(f.x + m * f.ldx + k0 + k + j), scales[m], inverses[m])
                                        : p.A[m * p.lda + k0 + k + j];
                    v |= (uint32_t)(uint8_t)q << (8 * j);
                }
            *reinterpret_cast<uint32_t*>(tokens + i) = v;
        }
        __syncthreads();
        if (n0 < p.N) {
            const int8_t* row[kChannels];
#pragma unroll
            for (int c = 0; c < kChannels; ++c) row[c] = p.B + (int64_t)min(n0 + c, p.N - 1) * p.ldb + k0;
            const int whole = len & ~15;
#pragma unroll 2
            for (int k = lane * 16; k < whole; k += 512) {
                int4 w[kChannels];
#pragma unroll
                for (int c = 0; c < kChannels; ++c) w[c] = load16<ALIGN>(row[c] + k);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int4 t = *reinterpret_cast<const int4*>(tokens + m * seg + k);
#pragma unroll
                    for (int c = 0; c < kChannels; ++c) acc[c][m] = dot16(w[c], t, acc[c][m]);
                }
            }
            if (lane < len - whole)  // the row's last bytes, one a lane
#pragma unroll
                for (int c = 0; c < kChannels; ++c)
#pragma unroll
                    for (int m = 0; m < MT; ++m) acc[c][m] += (int)row[c][whole + lane] * (int)tokens[m * seg + whole + lane];
        }
        __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < kChannels; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[c][m]);
            const int n = n0 + c;
            if (lane == (c * MT + m) % 32 && n < p.N && m < p.M)
                p.C[m * p.ldc + n] = i8_finish(sum, FUSED ? scales[m] : p.a_scale[m], p.b_scale[n], p.bias != nullptr,
                                               p.bias ? p.bias[n] : 0.0f, p.relu);
        }
}

template <int MT, int ALIGN, bool FUSED>
int launch_few(const FewArgs& f, cudaStream_t s) {
    const unsigned grid = (unsigned)((f.p.N + kFewThreads / 32 * kChannels - 1) / (kFewThreads / 32 * kChannels));
    const size_t smem = (size_t)MT * ((std::min(f.p.K, kSegment) + 15) & ~15);
    if (smem > 48 * 1024 && cudaFuncSetAttribute(gemm_i8_few_kernel<MT, ALIGN, FUSED>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, MT * kSegment) != cudaSuccess)
        return set_status(JST_ERR_CUDA, "cudaFuncSetAttribute(gemm_i8_few_kernel) failed");
    ProfScope prof(s, KID_GEMM_I8);
    if (launch_dependent(gemm_i8_few_kernel<MT, ALIGN, FUSED>, dim3(grid), dim3(kFewThreads), smem, s, f) != cudaSuccess)
        return set_status(JST_ERR_CUDA, "gemm_i8_few_kernel launch failed");
    return JST_OK;
}

template <bool FUSED>
int run_few(const FewArgs& f, cudaStream_t s) {
    const bool al = (reinterpret_cast<uintptr_t>(f.p.B) & 15) == 0 && (f.p.N == 1 || (f.p.ldb & 15) == 0);
    if (f.p.M == 1) return al ? launch_few<1, 16, FUSED>(f, s) : launch_few<1, 1, FUSED>(f, s);
    if (f.p.M == 2) return al ? launch_few<2, 16, FUSED>(f, s) : launch_few<2, 1, FUSED>(f, s);
    if (f.p.M <= 4) return al ? launch_few<4, 16, FUSED>(f, s) : launch_few<4, 1, FUSED>(f, s);
    return al ? launch_few<8, 16, FUSED>(f, s) : launch_few<8, 1, FUSED>(f, s);
}

// K == 0: every sum is 0.
__global__ void empty_sums_kernel(const I8Args p) {
    for (int64_t m = blockIdx.y; m < p.M; m += gridDim.y)
        for (int64_t n = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; n < p.N; n += (int64_t)gridDim.x * blockDim.x)
            p.C[m * p.ldc + n] = i8_finish(0, 0.0f, 0.0f, p.bias != nullptr, p.bias ? p.bias[n] : 0.0f, p.relu);
}

int run_empty(const I8Args& p, cudaStream_t s) {
    ProfScope prof(s, KID_GEMM_I8);
    empty_sums_kernel<<<dim3((unsigned)std::min((p.N + 255) / 256, 1024), (unsigned)std::min(p.M, 1024)), 256, 0, s>>>(p);
    return JST_OK;
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

// Up to kFew tokens the product is a read of the weight, and dp4a keeps up
// with it; from there on the tensor cores' work a byte of weight is free.
constexpr int kFew = 8;
// Up to so many values every block of the product quantises the tokens itself;
// more are quantised once, by a launch of their own.
constexpr int64_t kFusedValues = 16384;

int run_gemm_i8(const I8Args& p, cudaStream_t s) {
    const int rc = p.K == 0 ? run_empty(p, s) : p.M <= kFew ? run_few<false>({p, nullptr, 0}, s) : gemm_i8_tc_run(p, s);
    return rc ? rc : launched("gemm_i8 launch failed");
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
    I8Args p{M, N, K, nullptr, 0, w, ldw, nullptr, w_scale, (epilogue & JST_EPI_BIAS) ? bias : nullptr,
             (epilogue & JST_EPI_RELU) ? 1 : 0, y, ldy};
    if (K == 0 || (M <= kFew && (int64_t)M * K <= kFusedValues)) {
        rc = K == 0 ? run_empty(p, s) : run_few<true>({p, x, ldx}, s);
        return rc ? rc : launched("linear_i8 launch failed");
    }
    const int64_t ldq = ((int64_t)K + 15) / 16 * 16;
    const size_t scale_bytes = ((size_t)M * 4 + 255) & ~size_t(255);
    void* ws = nullptr;
    rc = workspace_alloc(scale_bytes + (size_t)M * ldq, s, &ws);
    if (rc) return rc;
    float* scale = static_cast<float*>(ws);
    int8_t* q = static_cast<int8_t*>(ws) + scale_bytes;
    rc = run_quantize(x, ldx, M, K, q, ldq, scale, s);
    if (!rc) {
        p.A = q;
        p.lda = ldq;
        p.a_scale = scale;
        rc = run_gemm_i8(p, s);
    }
    const int frc = workspace_free(ws, s);
    return rc ? rc : frc ? frc : set_status(JST_OK, nullptr);
}
