// dropout.cu -- jst_dropout (declared in include/jstorch_dropout.h): y = x * s
// where the element's random word is at least T, 0 elsewhere, in one pass over
// the data with the mask made in registers.
//
// The words come from Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011): ten rounds of two 32 x 32 -> 64
// multiplications give four words per counter, so a thread owns the four
// consecutive elements of one counter, and forward and backward make the same
// words from (seed, offset, index).
//
// Bound by memory: 8 bytes an element, against 5 wide multiplications and
// about 8 other integer operations of the generator.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/jstorch_dropout.h"
#include "gemm_internal.h"

namespace jst {
namespace {

constexpr int kThreads = 256;

// The four words of counter (block, call) under `key`.
__device__ __forceinline__ uint4 philox4x32_10(uint64_t block, uint64_t call, uint64_t key) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)call, c3 = (uint32_t)(call >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)q;
        c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

struct DropoutArgs {
    const float* x;
    float* y;
    int64_t ldx, ldy, rows, cols;
    uint32_t threshold;
    float scale;  // 0 when p == 1: nothing is kept
    uint64_t seed, offset;
    const int64_t* step;
};

// A dropped element is 0 whatever x holds, so the mask selects; x and y may be
// one buffer, so neither is __restrict__ and each thread loads before it stores.
__device__ __forceinline__ float drop(float v, uint32_t word, const DropoutArgs& a) {
    return word >= a.threshold && a.scale != 0.0f ? v * a.scale : 0.0f;
}

// One row, or rows without gaps: group g holds elements 4g .. 4g + 3.  A thread
// has the loads of G groups in flight while it makes their words: 67108864
// elements take 105 us with one, 91 with two, 80.4 with four (6.7 TB/s, 1.02 of
// the measured copy rate); 65536 elements, 1.5 us with one, 2.0 with four, as
// fewer SMs have work.
// VEC: both buffers are 16-byte aligned.
template <bool VEC, int G>
__global__ void __launch_bounds__(kThreads) dropout_flat_kernel(const DropoutArgs a, int64_t n) {
    const uint64_t call = a.offset + (a.step ? (uint64_t)*a.step : 0ull);
    const int64_t groups = (n + 3) >> 2, whole = n >> 2;
    for (int64_t g0 = blockIdx.x * (int64_t)(kThreads * G) + threadIdx.x; g0 < groups;
         g0 += (int64_t)gridDim.x * (kThreads * G)) {
        float4 v[G];
        if (VEC)
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const int64_t g = g0 + i * kThreads;
                if (g < whole) v[i] = reinterpret_cast<const float4*>(a.x)[g];
            }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int64_t g = g0 + i * kThreads;
            if (g >= groups) break;
            const uint4 r = philox4x32_10((uint64_t)g, call, a.seed);
            if (VEC && g < whole) {
                v[i].x = drop(v[i].x, r.x, a);
                v[i].y = drop(v[i].y, r.y, a);
                v[i].z = drop(v[i].z, r.z, a);
                v[i].w = drop(v[i].w, r.w, a);
                reinterpret_cast<float4*>(a.y)[g] = v[i];
            } else {
                const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (4 * g + j < n) a.y[4 * g + j] = drop(a.x[4 * g + j], w[j], a);
            }
        }
    }
}

// Rows with gaps: the elements of a group may lie in two rows or more.
__global__ void __launch_bounds__(kThreads) dropout_rows_kernel(const DropoutArgs a, int64_t n) {
    const uint64_t call = a.offset + (a.step ? (uint64_t)*a.step : 0ull);
    const int64_t groups = (n + 3) >> 2;
    for (int64_t g = blockIdx.x * (int64_t)kThreads + threadIdx.x; g < groups; g += (int64_t)gridDim.x * kThreads) {
        const int64_t i = g << 2;
        const uint4 r = philox4x32_10((uint64_t)g, call, a.seed);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        int64_t row = i / a.cols, col = i - row * a.cols;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j < n) a.y[row * a.ldy + col] = drop(a.x[row * a.ldx + col], w[j], a);
            if (++col == a.cols) {
                col = 0;
                ++row;
            }
        }
    }
}

}  // namespace
}  // namespace jst

extern "C" int jst_dropout(const float* x, int64_t ldx, float* y, int64_t ldy, int64_t rows, int64_t cols, double p,
                           uint64_t seed, uint64_t offset, const int64_t* step, jst_stream_t stream) {
    using namespace jst;
    if (rows < 0 || cols < 0) return set_status(JST_ERR_ARG, "dropout: negative size");
    if (!(p >= 0.0 && p <= 1.0)) return set_status(JST_ERR_ARG, "dropout: p must be in [0, 1]");
    if (cols > 0 && rows > INT64_MAX / 8 / cols) return set_status(JST_ERR_ARG, "dropout: size exceeds 64 bits");
    if (rows > 0 && cols > 0) {
        if (!x || !y) return set_status(JST_ERR_ARG, "dropout: null pointer");
        if (rows > 1 && (ldx < cols || ldy < cols)) return set_status(JST_ERR_ARG, "dropout: pitch < cols");
        if (rows > 1 && (ldx > INT64_MAX / 8 / rows || ldy > INT64_MAX / 8 / rows))
            return set_status(JST_ERR_ARG, "dropout: size exceeds 64 bits");
        const bool same = x == y && (ldx == ldy || rows == 1);
        const ByteRows out = byte_rows(y, rows, cols, ldy, 4);
        if (!same && rows_overlap(byte_rows(x, rows, cols, ldx, 4), out))
            return set_status(JST_ERR_ARG, "dropout: x and y overlap");
        if (step && rows_overlap(byte_rows(step, 1, 1, 1, 8), out))
            return set_status(JST_ERR_ARG, "dropout: y overlaps step");
    }
    int rc = require_device();
    if (rc) return rc;
    if (rows == 0 || cols == 0) return set_status(JST_OK, nullptr);
    DropoutArgs a;
    a.x = x; a.y = y;
    a.ldx = ldx; a.ldy = ldy; a.rows = rows; a.cols = cols;
    a.threshold = p < 1.0 ? (uint32_t)(p * 4294967296.0) : 0u;
    a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    a.seed = seed; a.offset = offset; a.step = step;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t n = rows * cols, groups = (n + 3) >> 2;
    const bool gaps = rows > 1 && (ldx != cols || ldy != cols);
    const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
    const int g = !gaps && groups >= 8 * (int64_t)kThreads * sm_count() ? 4 : 1;  // two such blocks an SM
    const unsigned grid = (unsigned)std::min<int64_t>((groups + kThreads * g - 1) / (kThreads * g), 1 << 20);
    {
        ProfScope prof(s, KID_DROPOUT);
        if (gaps) dropout_rows_kernel<<<grid, kThreads, 0, s>>>(a, n);
        else if (g == 4 && vec) dropout_flat_kernel<true, 4><<<grid, kThreads, 0, s>>>(a, n);
        else if (g == 4) dropout_flat_kernel<false, 4><<<grid, kThreads, 0, s>>>(a, n);
        else if (vec) dropout_flat_kernel<true, 1><<<grid, kThreads, 0, s>>>(a, n);
        else dropout_flat_kernel<false, 1><<<grid, kThreads, 0, s>>>(a, n);
    }
    return cudaPeekAtLastError() == cudaSuccess ? set_status(JST_OK, nullptr)
                                                : set_status(JST_ERR_CUDA, "dropout launch failed");
}
