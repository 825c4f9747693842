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

// One block a row.  NV > 0: the row's values stay in registers, NV groups of
// four a thread, between the peak and the quantisation, so x is read once;
// NV == 0 (rows of more than 32768 values) reads it twice.  Bound by memory: 5
// bytes a value.  VEC: x and q rows allow 16- and 4-byte accesses.
// 8192 x 8192 in 61 us (5.5 TB/s; with conversions and a division near a half 76);
// 4096 x 1024 in 6.8, which a warp a row does not change.
template <int NV, bool VEC>
__global__ void __launch_bounds__(1024)
    quantize_rows_kernel(const float* __restrict__ x, int64_t ldx, int cols, int8_t* __restrict__ q, int64_t ldq,
                         float* __restrict__ scale) {
    __shared__ uint32_t part[32];
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    const int n = blockDim.x;
    const float* row = x + (int64_t)blockIdx.x * ldx;
    int8_t* out = q + (int64_t)blockIdx.x * ldq;
    auto fetch = [&](int k) {
        if (VEC && k + 4 <= cols) return __ldg(reinterpret_cast<const float4*>(row + k));
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (k < cols) v.x = row[k];
        if (k + 1 < cols) v.y = row[k + 1];
        if (k + 2 < cols) v.z = row[k + 2];
        if (k + 3 < cols) v.w = row[k + 3];
        return v;
    };
    auto put = [&](int k, float4 v, float s, float inv) {
        const uint32_t word = quantize4(v, s, inv);
        if (VEC && k + 4 <= cols) {
            *reinterpret_cast<uint32_t*>(out + k) = word;
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < cols) out[k + j] = (int8_t)(uint8_t)(word >> (8 * j));
    };
    float4 v[NV ? NV : 1];
    uint32_t m = 0;
    auto peak = [&](const float4& f) {
        m = max(max(max(m, abs_bits(f.x)), max(abs_bits(f.y), abs_bits(f.z))), abs_bits(f.w));
    };
    if (NV) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = fetch(4 * (threadIdx.x + i * n));
#pragma unroll
        for (int i = 0; i < NV; ++i) peak(v[i]);
    } else {
        for (int k = 4 * threadIdx.x; k < cols; k += 4 * n) peak(fetch(k));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < n / 32 ? part[threadIdx.x & 31] : 0u);
    const float s = row_scale(m), inv = row_inverse(s);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    if (NV) {
#pragma unroll
        for (int i = 0; i < NV; ++i) put(4 * (threadIdx.x + i * n), v[i], s, inv);
    } else {
        for (int k = 4 * threadIdx.x; k < cols; k += 4 * n) put(k, fetch(k), s, inv);
    }
}

// ------------------------------------------------------------ one token
// A warp takes CH rows of the weight and walks along K, 16 bytes a lane and
// row: one 16-byte piece of the token from shared memory meets CH pieces
// of the weight, 4 dp4a each.  The lanes' sums meet in one integer reduction,
// exact in any order.
// Bound by the weight's bytes; each is read once, and asked of DRAM (a prefetch
// into L2) before the block turns to the token or waits for the launch before.
// The token is held in shared memory kSegment values of K at a time.  NV > 0
// (K <= 1024 NV): it comes as fp32 values and every block quantises it itself,
// NV groups of four a thread.
// ALIGN: 16 when the weight's rows are 16-byte aligned.  Otherwise 1: a lane
// reads the aligned 4-byte words that hold its 16 bytes and shifts; a word that
// holds a byte of the row does not leave the memory block that the row is in.
// The rows are dealt to the blocks in turn, and the blocks are a multiple of the
// SMs: each SM reads as much (1024 x 8192: 5.8 us, packed into full blocks 6.2;
// 128 x 4096: 3.5 and 3.8).
// Two rows a warp and four pieces of each in flight: 8192 x 8192 in 15.7 us
// (4.3 TB/s; a row maximum of as many bytes takes 14.6), with one row 16.8 and
// with four 23.7; quantising the token here adds nothing, a launch of its own 4.
constexpr int kOneThreads = 256;
constexpr int CH = 2;
constexpr int kSegment = 8192;

struct OneArgs {
    I8Args p;        // NV > 0: A and a_scale are unused
    const float* x;  // NV > 0: [K] fp32
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

template <int ALIGN, int NV>
__global__ void __launch_bounds__(kOneThreads) gemm_i8_one_kernel(const OneArgs f) {
    __shared__ __align__(16) int8_t token[kSegment];
    __shared__ uint32_t part[kOneThreads / 32];
    const I8Args& p = f.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = (warp * gridDim.x + blockIdx.x) * CH;
    if (n0 < p.N)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int8_t* row = p.B + (int64_t)min(n0 + c, p.N - 1) * p.ldb;
            for (int k = lane * 128; k < p.K; k += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + k));
        }
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    float scale = 0.0f;
    if (NV) {
        const bool vec = (reinterpret_cast<uintptr_t>(f.x) & 15) == 0;
        float4 v[NV ? NV : 1];
        uint32_t peak = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = 4 * (threadIdx.x + i * kOneThreads);
            if (vec && k + 4 <= p.K) {
                v[i] = __ldg(reinterpret_cast<const float4*>(f.x + k));
            } else {
                v[i].x = k < p.K ? __ldg(f.x + k) : 0.0f;
                v[i].y = k + 1 < p.K ? __ldg(f.x + k + 1) : 0.0f;
                v[i].z = k + 2 < p.K ? __ldg(f.x + k + 2) : 0.0f;
                v[i].w = k + 3 < p.K ? __ldg(f.x + k + 3) : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            peak = max(max(max(peak, abs_bits(v[i].x)), max(abs_bits(v[i].y), abs_bits(v[i].z))), abs_bits(v[i].w));
        peak = __reduce_max_sync(0xffffffffu, peak);
        if (lane == 0) part[warp] = peak;
        __syncthreads();
        scale = row_scale(__reduce_max_sync(0xffffffffu, lane < kOneThreads / 32 ? part[lane] : 0u));
        const float inv = row_inverse(scale);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = 4 * (threadIdx.x + i * kOneThreads);
            if (k < p.K)
                *reinterpret_cast<uint32_t*>(token + k) = quantize4(v[i], scale, inv);
        }
    } else {
        scale = __ldg(p.a_scale);
    }
    int acc[CH] = {};
    for (int k0 = 0; k0 < p.K; k0 += kSegment) {
        const int len = min(kSegment, p.K - k0);
        if (!NV)
            for (int k = threadIdx.x * 4; k < len; k += kOneThreads * 4) {
                uint32_t v = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k + j < len) v |= (uint32_t)(uint8_t)p.A[k0 + k + j] << (8 * j);
                *reinterpret_cast<uint32_t*>(token + k) = v;
            }
        __syncthreads();
        if (n0 < p.N) {
            const int8_t* row[CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) row[c] = p.B + (int64_t)min(n0 + c, p.N - 1) * p.ldb + k0;
            const int whole = len & ~15;
#pragma unroll(8 / CH)
            for (int k = lane * 16; k < whole; k += 512) {
                int4 w[CH];
#pragma unroll
                for (int c = 0; c < CH; ++c) w[c] = load16<ALIGN>(row[c] + k);
                const int4 t = *reinterpret_cast<const int4*>(token + k);
#pragma unroll
                for (int c = 0; c < CH; ++c) acc[c] = dot16(w[c], t, acc[c]);
            }
            if (lane < len - whole)  // the row's last bytes, one a lane
#pragma unroll
                for (int c = 0; c < CH; ++c) acc[c] += (int)row[c][whole + lane] * (int)token[whole + lane];
        }
        __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[c]), n = n0 + c;
        if (lane == c && n < p.N)
            p.C[n] = i8_finish(sum, scale, p.b_scale[n], p.bias != nullptr, p.bias ? p.bias[n] : 0.0f, p.relu);
    }
}

template <int ALIGN, int NV>
int launch_one(const OneArgs& f, cudaStream_t s) {
    constexpr int rows = kOneThreads / 32 * CH;
    const int sms = sm_count(), blocks = (f.p.N + rows - 1) / rows;
    const int even = std::min((blocks + sms - 1) / sms * sms, (f.p.N + CH - 1) / CH);
    ProfScope prof(s, KID_GEMM_I8);
    if (launch_dependent(gemm_i8_one_kernel<ALIGN, NV>, dim3((unsigned)even), dim3(kOneThreads), 0, s, f) != cudaSuccess)
        return set_status(JST_ERR_CUDA, "gemm_i8_one_kernel launch failed");
    return JST_OK;
}

template <int NV>
int run_one_nv(const OneArgs& f, cudaStream_t s) {
    const bool al = (reinterpret_cast<uintptr_t>(f.p.B) & 15) == 0 && (f.p.N == 1 || (f.p.ldb & 15) == 0);
    return al ? launch_one<16, NV>(f, s) : launch_one<1, NV>(f, s);
}

// x: the token in fp32, K <= kSegment; or null, and the token is in A.
int run_one(const I8Args& p, const float* x, cudaStream_t s) {
    const OneArgs f{p, x};
    if (!x) return run_one_nv<0>(f, s);
    return p.K <= 1024 ? run_one_nv<1>(f, s) : p.K <= 4096 ? run_one_nv<4>(f, s) : run_one_nv<8>(f, s);
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

// Rows and columns up to this: the kernels count in 32 bits and round up to tiles.
constexpr int kMost = 0x7fff0000;

int check_quantize(const float* x, int64_t ldx, int rows, int cols, const int8_t* q, int64_t ldq, const float* scale) {
    if (rows < 0 || cols < 0) return set_status(JST_ERR_ARG, "quantize_rows: negative size");
    if (rows > kMost || cols > kMost) return set_status(JST_ERR_ARG, "quantize_rows: size > 0x7fff0000");
    if (rows == 0) return JST_OK;
    if (!scale || (cols > 0 && (!x || !q))) return set_status(JST_ERR_ARG, "quantize_rows: null pointer");
    if (rows > 1 && (ldx < cols || ldq < cols)) return set_status(JST_ERR_ARG, "quantize_rows: pitch < cols");
    if (rows > 1 && (ldx > INT64_MAX / 8 / rows || ldq > INT64_MAX / 8 / rows))
        return set_status(JST_ERR_ARG, "quantize_rows: size exceeds 64 bits");
    if (cols == 0) return JST_OK;
    const ByteRows in = byte_rows(x, rows, cols, ldx, 4), out = byte_rows(q, rows, cols, ldq, 1), scales = byte_rows(scale, 1, rows, rows, 4);
    if (rows_overlap(out, in) || rows_overlap(scales, in) || rows_overlap(scales, out))
        return set_status(JST_ERR_ARG, "quantize_rows: an output overlaps another array");
    return JST_OK;
}

int run_quantize(const float* x, int64_t ldx, int rows, int cols, int8_t* q, int64_t ldq, float* scale, cudaStream_t s) {
    if (rows == 0) return set_status(JST_OK, nullptr);
    const bool vec = ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && (rows == 1 || (ldx & 3) == 0)) &&
                     ((reinterpret_cast<uintptr_t>(q) & 3) == 0 && (rows == 1 || (ldq & 3) == 0));
    // Groups of four values: few rows get a thread for each (a row's latency is
    // what counts), many rows up to eight a thread.
    const int groups = (cols + 3) / 4;
    int threads = std::min(rows < 2 * sm_count() ? 1024 : 256, std::max(32, (groups + 31) / 32 * 32));
    int nv = (groups + threads - 1) / threads;
    if (nv > 8) {
        threads = 1024;
        nv = (groups + threads - 1) / threads;
    }
    auto go = [&](auto kernel) { return launch_dependent(kernel, dim3((unsigned)rows), dim3(threads), 0, s, x, ldx, cols, q, ldq, scale); };
    {
        ProfScope prof(s, KID_QUANT);
        const cudaError_t e = nv <= 1   ? (vec ? go(quantize_rows_kernel<1, true>) : go(quantize_rows_kernel<1, false>))
                              : nv <= 2 ? (vec ? go(quantize_rows_kernel<2, true>) : go(quantize_rows_kernel<2, false>))
                              : nv <= 4 ? (vec ? go(quantize_rows_kernel<4, true>) : go(quantize_rows_kernel<4, false>))
                              : nv <= 8 ? (vec ? go(quantize_rows_kernel<8, true>) : go(quantize_rows_kernel<8, false>))
                                        : (vec ? go(quantize_rows_kernel<0, true>) : go(quantize_rows_kernel<0, false>));
        if (e != cudaSuccess) return set_status(JST_ERR_CUDA, "quantize_rows launch failed");
    }
    return launched("quantize_rows launch failed");
}

// The parts of a descriptor that jst_gemm_i8 and jst_linear_i8 share.
int check_product(int M, int N, int K, int64_t ldb, const void* B, const float* b_scale, const float* bias,
                  int epilogue, const float* C, int64_t ldc) {
    if (M < 0 || N < 0 || K < 0) return set_status(JST_ERR_ARG, "gemm_i8: negative size");
    if (M > kMost || N > kMost) return set_status(JST_ERR_ARG, "gemm_i8: size > 0x7fff0000");
    if (K > 131071) return set_status(JST_ERR_ARG, "gemm_i8: K > 131071 (the sum could exceed 32 bits)");
    if (epilogue < JST_EPI_NONE || epilogue > JST_EPI_BIAS_RELU) return set_status(JST_ERR_ARG, "gemm_i8: unknown epilogue");
    if (M == 0 || N == 0) return JST_OK;
    if ((epilogue & JST_EPI_BIAS) && !bias) return set_status(JST_ERR_ARG, "gemm_i8: bias epilogue without a bias pointer");
    if (!C || !b_scale || (K > 0 && !B)) return set_status(JST_ERR_ARG, "gemm_i8: null pointer");
    if ((M > 1 && ldc < N) || (N > 1 && K > 0 && ldb < K)) return set_status(JST_ERR_ARG, "gemm_i8: pitch too small");
    if ((M > 1 && ldc > INT64_MAX / 8 / M) || (N > 1 && ldb > INT64_MAX / 8 / N))
        return set_status(JST_ERR_ARG, "gemm_i8: size exceeds 64 bits");
    const ByteRows out = byte_rows(C, M, N, ldc, 4);
    if (rows_overlap(out, byte_rows(B, N, K, ldb, 1)))
        return set_status(JST_ERR_ARG, "gemm_i8: C overlaps the weight");
    if (rows_overlap(out, byte_rows(b_scale, 1, N, N, 4)) ||
        ((epilogue & JST_EPI_BIAS) && rows_overlap(out, byte_rows(bias, 1, N, N, 4))))
        return set_status(JST_ERR_ARG, "gemm_i8: C overlaps the channels' scales or bias");
    return JST_OK;
}

// One row beyond kSegment, which run_one walks in pieces behind barriers, is
// faster on the tensor cores where the operands are read in place and fill some
// SMs (4096 x 65536: 91 us against 49, 16384 x 12288: 45 and 37, 1024 x 12288: 14.0
// and 12.7, 128 x 12288: 8.4 and 11.8).
int run_gemm_i8(const I8Args& p, cudaStream_t s) {
    const bool one = p.M == 1 && !(p.K > kSegment && p.N >= 1024 && gemm_i8_tc_in_place(p));
    const int rc = p.K == 0 ? run_empty(p, s) : one ? run_one(p, nullptr, s) : gemm_i8_tc_run(p, s);
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
        const ByteRows out = byte_rows(d->C, d->M, d->N, d->ldc, 4);
        if (rows_overlap(out, byte_rows(d->A, d->M, d->K, d->lda, 1)))
            return set_status(JST_ERR_ARG, "gemm_i8: C overlaps A");
        if (rows_overlap(out, byte_rows(d->a_scale, 1, d->M, d->M, 4)))
            return set_status(JST_ERR_ARG, "gemm_i8: C overlaps the tokens' scales");
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
        if (rows_overlap(byte_rows(y, M, N, ldy, 4), byte_rows(x, M, K, ldx, 4)))
            return set_status(JST_ERR_ARG, "linear_i8: y overlaps x");
    }
    rc = require_device();
    if (rc) return rc;
    if (M == 0 || N == 0) return set_status(JST_OK, nullptr);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    I8Args p{M, N, K, nullptr, 0, w, ldw, nullptr, w_scale, (epilogue & JST_EPI_BIAS) ? bias : nullptr,
             (epilogue & JST_EPI_RELU) ? 1 : 0, y, ldy};
    if (K == 0 || (M == 1 && K <= kSegment)) {
        rc = K == 0 ? run_empty(p, s) : run_one(p, x, s);
        return rc ? rc : launched("linear_i8 launch failed");
    }
    if (M > 1 && gemm_i8_tc_takes_fp32(p)) {
        rc = gemm_i8_tc_run_fp32(p, x, ldx, s);
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
