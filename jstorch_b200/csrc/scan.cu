// scan.cu -- jst_scan_forward / jst_scan_backward (declared in
// include/jstorch_scan.h): the gated linear recurrence
//   z = sigmoid(a)   n = tanh(c) or c   h_t = z_t h_{t-1} + (1 - z_t) n_t
// and its gradients
//   G_t = dout_t + z_{t+1} G_{t+1}      (last step: dout_t + dh_n)
//   da_t = G_t (h_{t-1} - n_t) z_t (1 - z_t)
//   dc_t = G_t (1 - z_t) (1 - n_t^2 or 1)      dh0 = z_0 G_0
// Both are first-order recurrences  e' = A e + B  along one channel:
//   forward  e = h,                A = z,  B = (1 - z) n
//   backward e_t = z_{t+1} G_{t+1} (what the later steps hand back; dh_n at
//            the last one),  A = z_t,  B = z_t dout_t
// A step outside its sequence is A = 1, B = 0, chosen by comparison, so what
// the gates hold there (infinities and NaN too) does not matter.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/jstorch_scan.h"
#include "gemm_internal.h"

namespace jst {
namespace {

struct ScanArgs {
    const float* gates; int64_t ld_gates;
    const float* h0;
    const int32_t* lengths;
    const float* out_in; int64_t ld_out;  // backward: the forward's out
    const float* dout; int64_t ld_dout;
    const float* dh_n;
    float* out;      // forward
    float* h_n;      // forward
    float* dgates; int64_t ld_dgates;
    float* dh0;
    int seq, batch, hidden, reverse;
};

// sigmoid(a) and 1 - sigmoid(a) from one exponential of -|a|: neither loses
// digits where it is small.
__device__ __forceinline__ void gate(float a, float& z, float& rest) {
    const float e = expf(-fabsf(a));
    const float big = __fdividef(1.0f, 1.0f + e), small = e * big;
    z = a >= 0.0f ? big : small;
    rest = a >= 0.0f ? small : big;
}

template <bool TANH>
__device__ __forceinline__ float candidate(float c) {
    return TANH ? tanhf(c) : c;
}

// One thread per channel walks the time axis, K steps' loads at a time.
constexpr int kSerialThreads = 128;
constexpr int kSerialSteps = 8;

template <bool TANH>
__global__ void __launch_bounds__(kSerialThreads) scan_forward_serial_kernel(const ScanArgs p) {
    const int64_t channels = (int64_t)p.batch * p.hidden;
    const int64_t ch = blockIdx.x * (int64_t)kSerialThreads + threadIdx.x;
    if (ch >= channels) return;
    const int b = (int)(ch / p.hidden), j = (int)(ch - (int64_t)b * p.hidden);
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.seq) : p.seq;
    const int64_t step_g = (int64_t)p.batch * p.ld_gates, step_o = (int64_t)p.batch * p.ld_out;
    const float* g = p.gates + b * p.ld_gates + j;
    float* o = p.out + b * p.ld_out + j;
    float h = p.h0 ? p.h0[ch] : 0.0f;
    for (int s0 = 0; s0 < p.seq; s0 += kSerialSteps) {
        float a[kSerialSteps], c[kSerialSteps];
#pragma unroll
        for (int i = 0; i < kSerialSteps; ++i) {
            const int s = s0 + i, t = p.reverse ? p.seq - 1 - s : s;
            const bool in = s < p.seq && t < len;
            a[i] = in ? g[t * step_g] : 0.0f;
            c[i] = in ? g[t * step_g + p.hidden] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kSerialSteps; ++i) {
            const int s = s0 + i, t = p.reverse ? p.seq - 1 - s : s;
            if (s >= p.seq) break;
            if (t < len) {
                float z, rest;
                gate(a[i], z, rest);
                h = fmaf(z, h, rest * candidate<TANH>(c[i]));
            }
            o[t * step_o] = t < len ? h : 0.0f;
        }
    }
    if (p.h_n) p.h_n[ch] = h;
}

template <bool TANH>
__global__ void __launch_bounds__(kSerialThreads) scan_backward_serial_kernel(const ScanArgs p) {
    const int64_t channels = (int64_t)p.batch * p.hidden;
    const int64_t ch = blockIdx.x * (int64_t)kSerialThreads + threadIdx.x;
    if (ch >= channels) return;
    const int b = (int)(ch / p.hidden), j = (int)(ch - (int64_t)b * p.hidden);
    const int len = p.lengths ? min(max(p.lengths[b], 0), p.seq) : p.seq;
    const int64_t step_g = (int64_t)p.batch * p.ld_gates, step_o = (int64_t)p.batch * p.ld_out;
    const int64_t step_d = (int64_t)p.batch * p.ld_dout, step_dg = (int64_t)p.batch * p.ld_dgates;
    const float* g = p.gates + b * p.ld_gates + j;
    const float* o = p.out_in + b * p.ld_out + j;
    const float* d = p.dout ? p.dout + b * p.ld_dout + j : nullptr;
    float* dg = p.dgates + b * p.ld_dgates + j;
    const float h_first = p.h0 ? p.h0[ch] : 0.0f;
    const int first = p.reverse ? len - 1 : 0;  // the step that started from h0
    float e = p.dh_n ? p.dh_n[ch] : 0.0f;
    for (int s = 0; s < p.seq; ++s) {
        const int t = p.reverse ? s : p.seq - 1 - s;
        float da = 0.0f, dc = 0.0f;
        if (t < len) {
            float z, rest;
            gate(g[t * step_g], z, rest);
            const float n = candidate<TANH>(g[t * step_g + p.hidden]);
            const float h = t == first ? h_first : o[(p.reverse ? t + 1 : t - 1) * step_o];
            const float G = e + (d ? d[t * step_d] : 0.0f);
            da = G * ((h - n) * (z * rest));
            dc = G * (TANH ? rest * (1.0f - n * n) : rest);
            e = z * G;
        }
        dg[t * step_dg] = da;
        dg[t * step_dg + p.hidden] = dc;
    }
    if (p.dh0) p.dh0[ch] = e;
}

int check(const char* what, const ScanArgs& p, int candidate, bool backward) {
    if (p.seq < 0 || p.batch < 0 || p.hidden < 0) return set_status(JST_ERR_ARG, "scan: negative size");
    if (candidate != JST_SCAN_TANH && candidate != JST_SCAN_IDENTITY)
        return set_status(JST_ERR_ARG, "scan: unknown candidate function");
    const int64_t rows = (int64_t)p.seq * p.batch, H = p.hidden;
    if (rows == 0 || H == 0) return JST_OK;
    const int64_t most = INT64_MAX / 8 / rows;
    if (p.ld_gates < 2 * H || p.ld_out < H) return set_status(JST_ERR_ARG, "scan: pitch too small");
    if (p.ld_gates > most || p.ld_out > most) return set_status(JST_ERR_ARG, "scan: size exceeds 64 bits");
    if (!p.gates) return set_status(JST_ERR_ARG, "scan: null gates");
    const int64_t span_g = ((rows - 1) * p.ld_gates + 2 * H) * 4, span_o = ((rows - 1) * p.ld_out + H) * 4;
    const int64_t state = (int64_t)p.batch * H * 4;
    if (!backward) {
        if (!p.out) return set_status(JST_ERR_ARG, "scan: null out");
        if (ranges_overlap(p.out, span_o, p.gates, span_g) || (p.h0 && ranges_overlap(p.out, span_o, p.h0, state)) ||
            (p.h_n && (ranges_overlap(p.h_n, state, p.gates, span_g) || ranges_overlap(p.h_n, state, p.out, span_o))) ||
            (p.h_n && p.h0 && p.h_n != p.h0 && ranges_overlap(p.h_n, state, p.h0, state)))
            return set_status(JST_ERR_ARG, "scan: an output overlaps an input");
        return JST_OK;
    }
    if (!p.out_in || !p.dgates) return set_status(JST_ERR_ARG, "scan backward: null out or dgates");
    if (p.ld_dgates < 2 * H || (p.dout && p.ld_dout < H)) return set_status(JST_ERR_ARG, "scan backward: pitch too small");
    if (p.ld_dgates > most || (p.dout && p.ld_dout > most)) return set_status(JST_ERR_ARG, "scan backward: size exceeds 64 bits");
    const int64_t span_dg = ((rows - 1) * p.ld_dgates + 2 * H) * 4, span_d = p.dout ? ((rows - 1) * p.ld_dout + H) * 4 : 0;
    const struct { const void* at; int64_t bytes; } in[] = {
        {p.gates, span_g}, {p.out_in, span_o}, {p.dout, span_d}, {p.h0, state}, {p.dh_n, state}};
    for (const auto& i : in) {
        if (!i.at) continue;
        if (ranges_overlap(p.dgates, span_dg, i.at, i.bytes)) return set_status(JST_ERR_ARG, "scan backward: dgates overlaps an input");
        if (p.dh0 && !(i.at == p.dh0 && i.at == p.dh_n) && ranges_overlap(p.dh0, state, i.at, i.bytes))
            return set_status(JST_ERR_ARG, "scan backward: dh0 overlaps an input");
    }
    if (p.dh0 && ranges_overlap(p.dh0, state, p.dgates, span_dg))
        return set_status(JST_ERR_ARG, "scan backward: dh0 overlaps dgates");
    (void)what;
    return JST_OK;
}

// No step at all: the state (or its gradient) passes through.
int pass_state(float* dst, const float* src, int64_t n, cudaStream_t s) {
    if (!dst || n == 0 || dst == src) return set_status(JST_OK, nullptr);
    const cudaError_t e = src ? cudaMemcpyAsync(dst, src, (size_t)n * 4, cudaMemcpyDeviceToDevice, s)
                              : cudaMemsetAsync(dst, 0, (size_t)n * 4, s);
    if (e == cudaSuccess) return set_status(JST_OK, nullptr);
    cudaGetLastError();
    return set_status(JST_ERR_CUDA, "scan: state copy");
}

int launched(const char* what) {
    return cudaPeekAtLastError() == cudaSuccess ? set_status(JST_OK, nullptr) : set_status(JST_ERR_CUDA, what);
}

}  // namespace
}  // namespace jst

extern "C" int jst_scan_forward(const float* gates, int64_t ld_gates, int seq, int batch, int hidden, const float* h0,
                                const int32_t* lengths, int reverse, int candidate, float* out, int64_t ld_out,
                                float* h_n, jst_stream_t stream) {
    using namespace jst;
    ScanArgs p{};
    p.gates = gates; p.ld_gates = ld_gates;
    p.h0 = h0; p.lengths = lengths;
    p.out = out; p.ld_out = ld_out; p.h_n = h_n;
    p.seq = seq; p.batch = batch; p.hidden = hidden; p.reverse = reverse != 0;
    int rc = check("scan", p, candidate, false);
    if (rc) return rc;
    rc = require_device();
    if (rc) return rc;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t channels = (int64_t)batch * hidden;
    if (channels == 0) return set_status(JST_OK, nullptr);
    if (seq == 0) return pass_state(h_n, h0, channels, s);
    {
        ProfScope prof(s, KID_SCAN);
        const unsigned grid = (unsigned)((channels + kSerialThreads - 1) / kSerialThreads);
        if (candidate == JST_SCAN_TANH) scan_forward_serial_kernel<true><<<grid, kSerialThreads, 0, s>>>(p);
        else scan_forward_serial_kernel<false><<<grid, kSerialThreads, 0, s>>>(p);
    }
    return launched("scan launch failed");
}

extern "C" int jst_scan_backward(const float* gates, int64_t ld_gates, int seq, int batch, int hidden, const float* h0,
                                 const int32_t* lengths, int reverse, int candidate, const float* out, int64_t ld_out,
                                 const float* dout, int64_t ld_dout, const float* dh_n, float* dgates,
                                 int64_t ld_dgates, float* dh0, jst_stream_t stream) {
    using namespace jst;
    ScanArgs p{};
    p.gates = gates; p.ld_gates = ld_gates;
    p.h0 = h0; p.lengths = lengths;
    p.out_in = out; p.ld_out = ld_out;
    p.dout = dout; p.ld_dout = ld_dout; p.dh_n = dh_n;
    p.dgates = dgates; p.ld_dgates = ld_dgates; p.dh0 = dh0;
    p.seq = seq; p.batch = batch; p.hidden = hidden; p.reverse = reverse != 0;
    int rc = check("scan backward", p, candidate, true);
    if (rc) return rc;
    rc = require_device();
    if (rc) return rc;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t channels = (int64_t)batch * hidden;
    if (channels == 0) return set_status(JST_OK, nullptr);
    if (seq == 0) return pass_state(dh0, dh_n, channels, s);
    {
        ProfScope prof(s, KID_SCAN);
        const unsigned grid = (unsigned)((channels + kSerialThreads - 1) / kSerialThreads);
        if (candidate == JST_SCAN_TANH) scan_backward_serial_kernel<true><<<grid, kSerialThreads, 0, s>>>(p);
        else scan_backward_serial_kernel<false><<<grid, kSerialThreads, 0, s>>>(p);
    }
    return launched("scan backward launch failed");
}
