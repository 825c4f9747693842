// scan.cu -- jst_scan_forward / jst_scan_backward (declared in
// include/jstorch_scan.h): the gated linear recurrence
//   z = sigmoid(a)   n = tanh(c) or c   h_t = z_t h_{t-1} + (1 - z_t) n_t
// and its gradients
//   G_t = dout_t + z_{t+1} G_{t+1}      (last step: dout_t + dh_n)
//   da_t = G_t (h_{t-1} - n_t) z_t (1 - z_t)
//   dc_t = G_t (1 - z_t) (dn/dc: 1 - n_t^2 or 1)      dh0 = z_0 G_0
// Both are first-order recurrences  e' = A e + B  along one channel:
//   forward  e = h,                A = z,  B = (1 - z) n
//   backward e_t = z_{t+1} G_{t+1} (what the later steps hand back; dh_n at
//            the last one),  A = z_t,  B = z_t dout_t
// A step outside its sequence is A = 1, B = 0, chosen by comparison, so what
// the gates hold there (infinities and NaN too) does not matter.
//
// Bytes a step and channel: forward 8 read, 4 written; backward 16 read, 8
// written; nothing but the outputs is kept for the backward pass, which makes
// the gates again.  Reached on a B200 (tanh): 2048 x 16 x 1024 forward 81 us
// (5.0 TB/s, 0.76 of the measured copy rate), backward 142 us (5.7 TB/s, 0.86);
// 65536 x 1 x 1024, identity, 189 us (4.3 TB/s) and 289 us (5.6 TB/s), where
// one tile's rounds follow each other.  Forward, what is left is issue slots:
// 39 instructions for 12 bytes.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "../../include/jstorch_scan.h"
#include "gemm_internal.h"
#include "ptx.cuh"

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
    uint32_t* err;
};

// V adjacent channels of one step.  Pairs go through the two-wide fp32
// instructions: with a few loads, one exponential and one reciprocal a gate the
// issue slots are what limits an SM here, and a pair takes one slot for both.
template <int V>
struct F {
    float v[V];
};
__device__ __forceinline__ uint64_t pack(const F<2>& a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v[0]), "f"(a.v[1]));
    return r;
}
__device__ __forceinline__ F<2> unpack(uint64_t a) {
    F<2> r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.v[0]), "=f"(r.v[1]) : "l"(a));
    return r;
}
template <int V>
__device__ __forceinline__ F<V> all(float x) {
    F<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = x;
    return r;
}
template <int V>
__device__ __forceinline__ F<V> fma(const F<V>& a, const F<V>& b, const F<V>& c) {
    if constexpr (V == 2) {
        uint64_t r;
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack(a)), "l"(pack(b)), "l"(pack(c)));
        return unpack(r);
    } else {
        return {fmaf(a.v[0], b.v[0], c.v[0])};
    }
}
template <int V>
__device__ __forceinline__ F<V> operator*(const F<V>& a, const F<V>& b) {
    if constexpr (V == 2) {
        uint64_t r;
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack(a)), "l"(pack(b)));
        return unpack(r);
    } else {
        return {__fmul_rn(a.v[0], b.v[0])};
    }
}
template <int V>
__device__ __forceinline__ F<V> operator+(const F<V>& a, const F<V>& b) {
    if constexpr (V == 2) {
        uint64_t r;
        asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack(a)), "l"(pack(b)));
        return unpack(r);
    } else {
        return {__fadd_rn(a.v[0], b.v[0])};
    }
}
template <int V>
__device__ __forceinline__ F<V> operator-(const F<V>& a) {  // folds into the operation that takes it
    F<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = -a.v[i];
    return r;
}

// exp(-TIMES x) as 2^(-x TIMES log2 e), TIMES 1 or 2 and |TIMES x| <= 127: the rounding
// error of that product (and of log2 e) is found by a fused multiply-add and put back
// to first order, so what is left is the 2^-22 of the power and a rounding.  Results
// below 2^-126 flush to 0.
template <int TIMES, int V>
__device__ __forceinline__ F<V> exp_minus(const F<V>& x) {
    const float log2e = TIMES * 1.44269502162933349609375f, log2e_rest = TIMES * 1.92596299112661746887e-8f;
    const F<V> t = x * all<V>(-log2e);
    F<V> r = fma(x, all<V>(-log2e), -t);
    r = fma(x, all<V>(-log2e_rest), r) * all<V>(0.693147180559945309f);
    F<V> e;
#pragma unroll
    for (int i = 0; i < V; ++i) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.v[i]) : "f"(t.v[i]));
    return fma(e, r, e);
}
template <int V>
__device__ __forceinline__ F<V> reciprocal(const F<V>& x) {
    F<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.v[i]) : "f"(x.v[i]));
    return r;
}
// Clamps that a NaN passes.
__device__ __forceinline__ float at_least(float x, float lo) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(lo));
    return r;
}
__device__ __forceinline__ float at_most(float x, float hi) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(hi));
    return r;
}

// z = 1 / (1 + e) and 1 - z = e z with e = exp(-a): neither loses digits where
// it is small.  The reciprocal takes one Newton step: its ulp leans to one side,
// and a state that is remembered for a thousand steps would add it up.  A gate
// whose z or 1 - z is no normal number (below 2^-126: |a| > 87.33) is closed or open
// altogether, and a closed one keeps nothing of a state of any size: a is clamped
// where 1 + e is above 2^126, whose reciprocal flushes to 0.  The residual q, at most 2^-22
// elsewhere, is 1 then, and rounded to an integer it is the 1 - z that e z lacks.
template <int V>
__device__ __forceinline__ void gate(const F<V>& a, F<V>& z, F<V>& rest) {
    constexpr float shift = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
    F<V> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x.v[i] = at_most(at_least(a.v[i], -88.0f), 127.0f);
    const F<V> e = exp_minus<1>(x), d = e + all<V>(1.0f), r = reciprocal(d), q = fma(-d, r, all<V>(1.0f));
    z = fma(r, q, r);
    rest = fma(e, z, (q + all<V>(shift)) + all<V>(-shift));
}

// n = tanh(c) = (1 - t) / (1 + t) of |c| with t = exp(-2 |c|), and below 0.6, where
// 1 - t would lose digits, c + c^3 P(c^2) with P of degree 4: the smallest largest
// relative error over (0, 0.6] (a linear programme over Chebyshev points; 0.047 of
// 2^-24, and 0.079 with the coefficients rounded to fp32).  slope: dn/dc, which is 4 t / (1 + t)^2 (where n
// rounds to 1 that keeps its digits, and 1 - n^2 has none) and below 0.6 1 - n^2.
template <bool TANH, bool SLOPE, int V>
__device__ __forceinline__ F<V> candidate(const F<V>& c, F<V>& slope) {
    if constexpr (!TANH) {
        return c;
    } else {
        F<V> x;
#pragma unroll
        for (int i = 0; i < V; ++i) x.v[i] = at_most(fabsf(c.v[i]), 60.0f);
        const F<V> t = exp_minus<2>(x), w = reciprocal(t + all<V>(1.0f));
        const F<V> far = (all<V>(1.0f) + -t) * w;
        const F<V> q = c * c;
        F<V> p = fma(q, all<V>(-0.005895157810300589f), all<V>(0.020795971155166626f));
        p = fma(p, q, all<V>(-0.053783830255270004f));
        p = fma(p, q, all<V>(0.13331924378871918f));
        p = fma(p, q, all<V>(-0.33333298563957214f));
        const F<V> near = fma(c * q, p, c);
        F<V> n;
#pragma unroll
        for (int i = 0; i < V; ++i) n.v[i] = fabsf(c.v[i]) < 0.6f ? near.v[i] : copysignf(far.v[i], c.v[i]);
        if (SLOPE) {
            const F<V> near_slope = fma(-near, near, all<V>(1.0f)), far_slope = t * all<V>(4.0f) * w * w;
#pragma unroll
            for (int i = 0; i < V; ++i) slope.v[i] = fabsf(c.v[i]) < 0.6f ? near_slope.v[i] : far_slope.v[i];
        }
        return n;
    }
}

// A product of z in (0, 1) underflows to 0 after some hundred steps, and 0 times
// an infinite state would be NaN where step by step it stays infinite: unless a z
// is 0, products are kept at 2^-149 at least, which is a rounding of theirs.
constexpr float kTiny = 1.40129846432481707e-45f;

template <int V>
__device__ __forceinline__ F<V> load(const char* p) {
    if constexpr (V == 2) {
        const float2 x = __ldg(reinterpret_cast<const float2*>(p));
        return {x.x, x.y};
    } else {
        return {__ldg(reinterpret_cast<const float*>(p))};
    }
}
// The backward's outputs are written past what it reads (64 x 64 x 1024: 18.5 us
// for 20.2); the forward's stay for their reader.
template <bool STREAM, int V>
__device__ __forceinline__ void store(char* p, const F<V>& x) {
    if constexpr (V == 2) {
        if (STREAM) __stcs(reinterpret_cast<float2*>(p), make_float2(x.v[0], x.v[1]));
        else *reinterpret_cast<float2*>(p) = make_float2(x.v[0], x.v[1]);
    } else {
        if (STREAM) __stcs(reinterpret_cast<float*>(p), x.v[0]);
        else *reinterpret_cast<float*>(p) = x.v[0];
    }
}

// Rows of one array as a warp walks them: the address of the tile's first
// channel at the pass's first step and the bytes of a step (both the same in
// all lanes, so steps are added in the uniform datapath), and this lane's
// bytes behind the tile's first channel.
struct Rows {
    char* base;
    int64_t step;
    uint32_t lane;

    __device__ __forceinline__ char* at(int64_t s) const { return base + s * step; }
};

// A warp's 32 * V channels and the direction of its pass.
template <bool BWD, int V>
struct Channels {
    bool mine;   // this lane's channels exist
    int64_t ch;  // its first one
    int lo, hi;  // steps of this pass inside its sequence: [lo, hi)
    uint32_t c;  // bytes from a row's a to its c
    Rows gates, out, dout, dgates;  // backward: out is h of the step that comes next in this pass

    __device__ __forceinline__ Rows rows(const ScanArgs& p, const float* x, int64_t ld, bool down, int64_t tile,
                                         int b, int j) const {
        const int b0 = (int)(tile / p.hidden), j0 = (int)(tile - (int64_t)b0 * p.hidden);
        Rows r;
        r.step = (down ? -4 : 4) * (p.batch * ld);
        r.base = const_cast<char*>(reinterpret_cast<const char*>(x + ((down ? p.seq - 1 : 0) * (int64_t)p.batch + b0) * ld + j0));
        r.lane = (uint32_t)(((b - b0) * ld + (j - j0)) * 4);
        return r;
    }
    // tile: the warp's first channel, the same in every lane
    __device__ __forceinline__ Channels(const ScanArgs& p, int64_t tile, int lane) {
        ch = tile + lane * V;
        const int64_t channels = (int64_t)p.batch * p.hidden;
        mine = ch < channels;
        const int64_t at = mine ? ch : channels - V;  // a lane past the end reads and writes nothing
        const int b = (int)(at / p.hidden), j = (int)(at - (int64_t)b * p.hidden);
        const int len = !mine ? 0 : p.lengths ? min(max(p.lengths[b], 0), p.seq) : p.seq;
        const bool down = BWD ? !p.reverse : p.reverse != 0;  // from the last step to the first
        lo = down ? p.seq - len : 0;
        hi = lo + len;
        c = (uint32_t)p.hidden * 4;
        gates = rows(p, p.gates, p.ld_gates, down, tile, b, j);
        if (BWD) {
            out = rows(p, p.out_in, p.ld_out, down, tile, b, j);
            out.base += out.step;
            dout = rows(p, p.dout, p.ld_dout, down, tile, b, j);
            dgates = rows(p, p.dgates, p.ld_dgates, down, tile, b, j);
        } else {
            out = rows(p, p.out, p.ld_out, down, tile, b, j);
        }
    }
    __device__ __forceinline__ F<V> state(const float* p) const {
        F<V> r;
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = mine && p ? p[ch + i] : 0.0f;
        return r;
    }
    __device__ __forceinline__ void set_state(float* p, const F<V>& x) const {
        if (mine && p)
#pragma unroll
            for (int i = 0; i < V; ++i) p[ch + i] = x.v[i];
    }
    // whether steps [s, s + n) are inside every lane's sequence
    __device__ __forceinline__ bool whole(int64_t s, int n) const {
        return __all_sync(0xffffffffu, s >= lo && s + n <= hi);
    }
    __device__ __forceinline__ bool in(int64_t s) const { return s >= lo && s < hi; }
};

// K steps of a lane's channels as they come from memory.
template <bool BWD, int V, int K>
struct Raw {
    F<V> a[K], c[K], h[BWD ? K : 1], d[BWD ? K : 1];

    template <bool ALL, bool DOUT>
    __device__ __forceinline__ void fetch_part(const Channels<BWD, V>& w, const F<V>& h_first, int64_t s0) {
        const char *g = w.gates.at(s0), *o = BWD ? w.out.at(s0) : nullptr, *d0 = BWD ? w.dout.at(s0) : nullptr;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const bool in = ALL || w.in(s0 + i);
            a[i] = in ? load<V>(g + w.gates.lane) : all<V>(0.0f);
            c[i] = in ? load<V>(g + w.c + w.gates.lane) : all<V>(0.0f);
            g += w.gates.step;
            if (BWD) {
                // the last step inside the sequence is the one that started from h0
                h[i] = !in ? all<V>(0.0f) : !ALL && s0 + i + 1 == w.hi ? h_first : load<V>(o + w.out.lane);
                d[i] = DOUT && in ? load<V>(d0 + w.dout.lane) : all<V>(0.0f);
                o += w.out.step;
                d0 += w.dout.step;
            }
        }
    }
    __device__ __forceinline__ void fetch(const ScanArgs& p, const Channels<BWD, V>& w, const F<V>& h_first, int64_t s0) {
        if (w.whole(s0, BWD ? K + 1 : K)) {
            if (!BWD || p.dout) fetch_part<true, BWD>(w, h_first, s0);
            else fetch_part<true, false>(w, h_first, s0);
        } else {
            if (!BWD || p.dout) fetch_part<false, BWD>(w, h_first, s0);
            else fetch_part<false, false>(w, h_first, s0);
        }
    }
};

// What the outputs of K steps need once the state before them is known:
// forward z and (1 - z) n; backward z, dout, and da and dc per unit of G.
template <bool BWD, int V, int K>
struct Steps {
    F<V> z[K], add[K], fa[BWD ? K : 1], fc[BWD ? K : 1];

    template <bool TANH>
    __device__ __forceinline__ void from(const Raw<BWD, V, K>& r, const Channels<BWD, V>& w, int64_t s0) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            F<V> rest;
            gate(r.a[i], z[i], rest);
            F<V> slope;
            const F<V> n = candidate<TANH, BWD>(r.c[i], slope);
            if (BWD) {
                fa[i] = (r.h[i] + -n) * (z[i] * rest);
                fc[i] = TANH ? rest * slope : rest;
                add[i] = r.d[i];
            } else {
                add[i] = rest * n;
            }
        }
        if (!w.whole(s0, K))
#pragma unroll
            for (int i = 0; i < K; ++i) {
                if (w.in(s0 + i)) continue;
                z[i] = all<V>(1.0f);  // the state passes over the step
                add[i] = all<V>(0.0f);
            }
    }
    // the steps as one pair (A, B): e -> A e + B
    __device__ __forceinline__ void fold(F<V>& A, F<V>& B) const {
        A = z[0];
        B = BWD ? z[0] * add[0] : add[0];
#pragma unroll
        for (int i = 1; i < K; ++i) {
            B = BWD ? z[i] * (B + add[i]) : fma(z[i], B, add[i]);
            A = A * z[i];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float least = kTiny;  // 0 where a z is
#pragma unroll
            for (int i = 0; i < K; ++i) least = fminf(least, z[i].v[v]);
            A.v[v] = fmaxf(A.v[v], least);
        }
    }
    template <bool ALL>
    __device__ __forceinline__ F<V> finish_part(F<V> e, int seq, const Channels<BWD, V>& w, int64_t s0) const {
        const Rows& r = BWD ? w.dgates : w.out;
        char* o = r.at(s0);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const bool in = ALL || w.in(s0 + i), exists = ALL || (w.mine && s0 + i < seq);
            if (BWD) {
                const F<V> G = e + add[i];
                const F<V> da = G * fa[i], dc = G * fc[i];
                if (exists) {
                    store<true>(o + r.lane, in ? da : all<V>(0.0f));
                    store<true>(o + w.c + r.lane, in ? dc : all<V>(0.0f));
                }
                e = z[i] * G;
            } else {
                e = fma(z[i], e, add[i]);
                if (exists) store<false>(o + r.lane, in ? e : all<V>(0.0f));
            }
            o += r.step;
        }
        return e;
    }
    // the state (or what is handed back) after the K steps; writes their outputs
    __device__ __forceinline__ F<V> finish(F<V> e, int seq, const Channels<BWD, V>& w, int64_t s0) const {
        return w.whole(s0, K) ? finish_part<true>(e, seq, w, s0) : finish_part<false>(e, seq, w, s0);
    }
};

// Zeros behind the sequences: the rows of steps [s, end), every stride-th run of K.
template <bool BWD, int V, int K>
__device__ __forceinline__ void write_zeros(const Channels<BWD, V>& w, int64_t s, int64_t end, int64_t stride, int seq) {
    const Rows& r = BWD ? w.dgates : w.out;
    for (; s < end; s += stride) {
        char* o = r.at(s);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (w.mine && s + i < seq) {
                store<BWD>(o + r.lane, all<V>(0.0f));
                if (BWD) store<BWD>(o + w.c + r.lane, all<V>(0.0f));
            }
            o += r.step;
        }
    }
}

// The warp's index, known to the compiler as the same in all lanes.
__device__ __forceinline__ int warp_index() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }

// ------------------------------------------------------------ short sequences
// One lane walks its channels' time axis, K steps' loads at a time.
constexpr int kSerialThreads = 128;

template <bool BWD, bool TANH, int V, int K>
__global__ void __launch_bounds__(kSerialThreads) scan_serial_kernel(const ScanArgs p) {
    const int64_t tile = (blockIdx.x * (int64_t)(kSerialThreads / 32) + warp_index()) * 32 * V;
    if (tile >= (int64_t)p.batch * p.hidden) return;
    const Channels<BWD, V> w(p, tile, threadIdx.x & 31);
    const F<V> h_first = w.state(p.h0);
    F<V> e = BWD ? w.state(p.dh_n) : h_first;
    for (int64_t s0 = 0; s0 < p.seq; s0 += K) {
        Raw<BWD, V, K> r;
        r.fetch(p, w, h_first, s0);
        Steps<BWD, V, K> st;
        st.template from<TANH>(r, w, s0);
        e = st.finish(e, p.seq, w, s0);
    }
    w.set_state(BWD ? p.dh0 : p.h_n, e);
}

// ------------------------------------------------------------ split along time
// A pair (A, B) stands for e -> A e + B.  K steps in a lane's registers fold
// into one pair; applying the pairs in the order of time to the state that the
// round starts from gives every lane the state before its own first step, and
// a second pass over the registers gives the outputs: the data are read once.
//   block    S warps over the same 32 * V channels (V a lane), K consecutive
//            steps a warp: one row segment of 32 * V floats a load;
//   cluster  C blocks over consecutive runs of S * K steps; each sends the
//            pair of its run to the others through distributed shared memory,
//            counted in by a barrier of the receiver (a cluster-wide barrier
//            a round would wait for every load and store in flight);
//   loop     until the time axis ends, C * S * K steps a round, with the next
//            round's loads in flight while this one is folded and written.
// Every order is fixed, so results repeat bit for bit.

// V channels' pair in shared memory.
template <int V>
struct __align__(8 * V) Pair {
    F<V> A, B;
};
// Store to the same place in block `rank` of the cluster; its barrier counts the bytes as they arrive.
template <int V>
__device__ __forceinline__ void send(Pair<V>* to, uint64_t* bar, int rank, const Pair<V>& v) {
    const uint32_t at = ptx::cluster_addr(ptx::smem_u32(to), rank), at_bar = ptx::cluster_addr(ptx::smem_u32(bar), rank);
    if constexpr (V == 2)
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at),
                     "r"(__float_as_uint(v.A.v[0])), "r"(__float_as_uint(v.A.v[1])), "r"(__float_as_uint(v.B.v[0])),
                     "r"(__float_as_uint(v.B.v[1])), "r"(at_bar)
                     : "memory");
    else
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(at),
                     "r"(__float_as_uint(v.A.v[0])), "r"(__float_as_uint(v.B.v[0])), "r"(at_bar)
                     : "memory");
}

constexpr int kMostBlocks = 16;  // of a cluster

template <bool BWD, bool TANH, int V, int S, int K, int BLOCKS>
__global__ void __launch_bounds__(32 * S, BLOCKS) scan_tiled_kernel(const ScanArgs p, int C) {
    __shared__ Pair<V> warps[2][S][32];   // the warps' folds, two rounds
    __shared__ Pair<V> blocks[2][kMostBlocks][32];  // the folds of the cluster's blocks, two rounds
    __shared__ uint64_t arrived[2];
    __shared__ uint32_t gave_up;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x % C);  // C divides the grid: the block's rank in its cluster
    const Channels<BWD, V> w(p, (blockIdx.x / C) * (int64_t)(32 * V), lane);
    const F<V> h_first = w.state(p.h0);
    F<V> carry = BWD ? w.state(p.dh_n) : h_first;
    const int64_t round_steps = (int64_t)C * S * K, my_first = (int64_t)(rank * S + warp) * K;
    // The rounds that some channel of the tile has steps in; the others, before
    // and behind, are zeros alone.  The same in all warps and blocks of the cluster.
    const int some_lo = __reduce_min_sync(0xffffffffu, w.lo < w.hi ? w.lo : p.seq);
    const int some_hi = __reduce_max_sync(0xffffffffu, w.lo < w.hi ? w.hi : 0);
    const int64_t begin = some_lo / round_steps * round_steps;
    const int64_t end = (some_hi + round_steps - 1) / round_steps * round_steps;
    Raw<BWD, V, K> raw;
    raw.fetch(p, w, h_first, begin + my_first);
    if (C > 1) {
        if (threadIdx.x == 0) {
            ptx::mbar_init(&arrived[0], 1);
            ptx::mbar_init(&arrived[1], 1);
            gave_up = 0;
            ptx::fence_barrier_init();
        }
        ptx::cluster_arrive();  // every block's barriers are set up before any block sends
        ptx::cluster_wait();
    }
    uint32_t round = 0;
    for (int64_t base = begin; base < end; base += round_steps, ++round) {
        const int parity = round & 1;
        const int64_t s0 = base + my_first;
        if (C > 1 && threadIdx.x == 0) ptx::mbar_arrive_expect_tx(&arrived[parity], (uint32_t)(C * 32 * sizeof(Pair<V>)));
        Steps<BWD, V, K> st;
        st.template from<TANH>(raw, w, s0);
        {
            Pair<V> mine;
            st.fold(mine.A, mine.B);
            warps[parity][warp][lane] = mine;
        }
        if (base + round_steps < end) raw.fetch(p, w, h_first, s0 + round_steps);
        // One barrier a round: a warp writes these places again two rounds on,
        // past the next barrier, which every warp reaches after reading them.
        __syncthreads();
        F<V> e = carry;  // the state before this block's run, then before this warp's
        if (C > 1) {
            if (warp == 0) {
                Pair<V> run = warps[parity][0][lane];
#pragma unroll
                for (int q = 1; q < S; ++q) {
                    const Pair<V> f = warps[parity][q][lane];
                    run.B = fma(f.A, run.B, f.B);
                    const F<V> A = f.A * run.A;
#pragma unroll
                    for (int v = 0; v < V; ++v)  // 0 where a factor is
                        run.A.v[v] = fmaxf(A.v[v], fminf(fminf(f.A.v[v], run.A.v[v]), kTiny));
                }
                // A block is two rounds ahead of another's reads of these places
                // only after that other has sent the round between: it has read them.
                for (int q = 0; q < C; ++q) send(&blocks[parity][rank][lane], &arrived[parity], q, run);
            }
            ptx::mbar_wait<true>(&arrived[parity], (round >> 1) & 1, &gave_up);
            for (int q = 0; q < C; ++q) {
                if (q == rank) e = carry;
                const Pair<V> f = blocks[parity][q][lane];
                carry = fma(f.A, carry, f.B);
            }
#pragma unroll
            for (int q = 0; q < S - 1; ++q) {
                if (q >= warp) break;
                const Pair<V> f = warps[parity][q][lane];
                e = fma(f.A, e, f.B);
            }
        } else {
#pragma unroll
            for (int q = 0; q < S; ++q) {
                if (q == warp) e = carry;
                const Pair<V> f = warps[parity][q][lane];
                carry = fma(f.A, carry, f.B);
            }
        }
        st.finish(e, p.seq, w, s0);
    }
    if (rank == 0 && warp == 0) w.set_state(BWD ? p.dh0 : p.h_n, carry);
    write_zeros<BWD, V, K>(w, my_first, begin, round_steps, p.seq);
    write_zeros<BWD, V, K>(w, std::max(end, begin) + my_first, p.seq, round_steps, p.seq);
    if (C > 1) {
        if (threadIdx.x == 0 && gave_up) atomicOr(p.err, gave_up);
        ptx::cluster_arrive();  // nobody leaves while another could still send to it
        ptx::cluster_wait();
    }
}

// The largest cluster that tests leave to the device (jst_test_scan_cluster).
std::atomic<int> test_cluster{kMostBlocks};

// Whether the device places the cluster of `cfg`, which is larger than the 8 that every GPU
// of the architecture guarantees: it takes a GPC with that many free SMs.  Asked once a
// device and kernel.
template <bool BWD, bool TANH, int V, int S, int K, int BLOCKS>
bool cluster_fits(const cudaLaunchConfig_t& cfg) {
    static std::atomic<int> known[64] = {};  // 1: yes, 2: no
    const auto kernel = scan_tiled_kernel<BWD, TANH, V, S, K, BLOCKS>;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    int answer = known[dev].load(std::memory_order_relaxed);
    if (answer == 0) {
        int clusters = 0;
        const bool fits = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                          cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0;
        if (!fits) cudaGetLastError();
        answer = fits ? 1 : 2;
        known[dev].store(answer, std::memory_order_relaxed);
    }
    return answer == 1 && (int)cfg.attrs[0].val.clusterDim.x <= test_cluster.load(std::memory_order_relaxed);
}

template <bool BWD, bool TANH, int V, int S, int K, int BLOCKS>
int launch_tiled(const ScanArgs& p, int C, cudaStream_t s) {
    const int64_t tiles = ((int64_t)p.batch * p.hidden + 32 * V - 1) / (32 * V);
    const auto kernel = scan_tiled_kernel<BWD, TANH, V, S, K, BLOCKS>;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(32 * S);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto clusters_of = [&](int c) {
        C = c;
        cfg.gridDim = dim3((unsigned)(tiles * c));
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)c;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    };
    clusters_of(C);
    if (C > 8 && !cluster_fits<BWD, TANH, V, S, K, BLOCKS>(cfg)) clusters_of(8);
    ProfScope prof(s, KID_SCAN);
    return cudaLaunchKernelEx(&cfg, kernel, p, C) == cudaSuccess
               ? JST_OK
               : set_status(JST_ERR_CUDA, "scan launch failed");
}

// Which kernel, and how the time axis is split.  Times in us, tanh, forward
// and backward, on a B200 (tile: the 32 * V channels of a warp).
//   * A few steps, or enough channels to fill the SMs by themselves: one lane
//     walks the axis (4 x 64 x 1024 [seq x batch x hidden]: 2.7 / 3.6, split
//     over warps 5.7 / 8.8; 16 x 64 x 1024: 5.4 / 6.8, split 6.1 / 10.1;
//     128 x 256 x 1024: 69 / 139, split 84 / 150).
//   * Many tiles of a short axis: small blocks, of which many fit an SM
//     (64 x 64 x 1024: 12.3 / 18.5, 33 x 70 x 1024: 11.3 / 14.4 in blocks of 2 warps x 8
//     steps; 4 x 4: 13.7 / 18.9, 12.7 / 16.4; 8 x 8: 15.1 / 24.8 for the first).
//   * Otherwise 64 steps a block and round, 8 a lane (2048 x 16 x 1024 forward
//     81, with 4 steps a lane 100; backward 4 warps x 8 steps 142, 8 x 8 149,
//     4 x 4 200), and where the tiles leave SMs empty, clusters that share a
//     tile's axis: forward 2 blocks fit an SM, backward 1 (4096 x 1 x 4096:
//     45 / 77 in clusters of 4 / 2, 94 / 122 without).
//   * Long sequences of different lengths: twice the clusters, as the tiles of the
//     longest outlast the others (2048 x 16 x 1024 with lengths drawn evenly:
//     65 / 110, 78 / 132 without; at 1000 x 64 x 256 it costs, 40 / 68 for 37 / 67).
//   * So few channels that even clusters of 8 blocks leave SMs empty: one
//     channel a lane, twice the tiles (65536 x 1 x 1024, identity: 189 / 289
//     against 240 / 428 with two), and where even those leave half the SMs empty,
//     clusters of 16 (20000 x 1 x 32, identity: 26.0 / 32.9 for 41.0 / 56.3; with
//     32 tiles they cost, 270 for 190, as fewer such clusters find room).
template <bool BWD, bool TANH, int V>
int run_scan(const ScanArgs& p, cudaStream_t s) {
    const int64_t channels = (int64_t)p.batch * p.hidden, tiles = (channels + 32 * V - 1) / (32 * V);
    const int sms = sm_count();
    if (p.seq <= 16 || channels >= 131072) {
        const int64_t grid = (tiles + kSerialThreads / 32 - 1) / (kSerialThreads / 32);
        if (grid > 0x7fffffff) return set_status(JST_ERR_ARG, "scan: too many channels");
        ProfScope prof(s, KID_SCAN);
        scan_serial_kernel<BWD, TANH, V, 4><<<(unsigned)grid, kSerialThreads, 0, s>>>(p);
        return JST_OK;
    }
    if (p.seq <= 64 && tiles >= 4 * sms) return launch_tiled<BWD, TANH, V, 2, 8, BWD ? 4 : 8>(p, 1, s);
    const bool uneven = p.lengths && p.seq > 1024;
    if (BWD && V == 2 && tiles >= sms && !uneven) return launch_tiled<BWD, TANH, V, 4, 8, 1>(p, 1, s);
    constexpr int blocks_per_sm = BWD && V == 2 ? 1 : 2;
    int C = 1;
    while (C < 8 && tiles * C * 2 <= sms * blocks_per_sm * (uneven ? 2 : 1) && p.seq > C * 64) C *= 2;
    if (C == 8 && tiles * 16 <= sms && p.seq > 8 * 64) C = 16;
    return launch_tiled<BWD, TANH, V, 8, 8, blocks_per_sm>(p, C, s);
}

// Whether the V = 2 kernels' 8-byte accesses are aligned.
bool pairs_ok(const ScanArgs& p) {
    if (p.hidden & 1) return false;
    const struct { const void* at; int64_t ld; } rows[] = {
        {p.gates, p.ld_gates}, {p.out_in, p.ld_out}, {p.out, p.ld_out}, {p.dout, p.ld_dout}, {p.dgates, p.ld_dgates}};
    for (const auto& r : rows)
        if (r.at && ((reinterpret_cast<uintptr_t>(r.at) & 7) || (r.ld & 1))) return false;
    return true;
}

template <bool BWD>
int dispatch(const ScanArgs& p, int candidate, cudaStream_t s) {
    const int64_t channels = (int64_t)p.batch * p.hidden;
    const bool few = p.seq > 16 && (channels + 63) / 64 * 8 <= sm_count();
    const bool two = pairs_ok(p) && !few;
    if (candidate == JST_SCAN_TANH) return two ? run_scan<BWD, true, 2>(p, s) : run_scan<BWD, true, 1>(p, s);
    return two ? run_scan<BWD, false, 2>(p, s) : run_scan<BWD, false, 1>(p, s);
}

int check(const ScanArgs& p, int candidate, bool backward) {
    if (p.seq < 0 || p.batch < 0 || p.hidden < 0) return set_status(JST_ERR_ARG, "scan: negative size");
    if (candidate != JST_SCAN_TANH && candidate != JST_SCAN_IDENTITY)
        return set_status(JST_ERR_ARG, "scan: unknown candidate function");
    const int64_t rows = (int64_t)p.seq * p.batch, H = p.hidden;
    if (rows == 0 || H == 0) return JST_OK;
    const int64_t most = INT64_MAX / 8 / rows;
    if (p.ld_gates < 2 * H || p.ld_out < H) return set_status(JST_ERR_ARG, "scan: pitch too small");
    // a warp's channels may lie in 32 rows: their distance is held in 32 bits
    const int64_t wide = 1 << 24;
    if (p.ld_gates >= wide || p.ld_out >= wide || (backward && (p.ld_dgates >= wide || (p.dout && p.ld_dout >= wide))))
        return set_status(JST_ERR_ARG, "scan: pitch >= 2^24");
    if (p.ld_gates > most || p.ld_out > most) return set_status(JST_ERR_ARG, "scan: size exceeds 64 bits");
    if (!p.gates) return set_status(JST_ERR_ARG, "scan: null gates");
    const int64_t state = (int64_t)p.batch * H;
    auto vector = [](const void* at, int64_t n) { return byte_rows(at, 1, n, n, 4); };
    auto matrix = [&](const void* at, int64_t cols, int64_t ld) { return byte_rows(at, rows, cols, ld, 4); };
    const ByteRows gates = matrix(p.gates, 2 * H, p.ld_gates), h0 = vector(p.h0, state), lengths = vector(p.lengths, p.batch);
    if (!backward) {
        if (!p.out) return set_status(JST_ERR_ARG, "scan: null out");
        const ByteRows out = matrix(p.out, H, p.ld_out), h_n = vector(p.h_n, state);
        if (rows_overlap(out, gates) || rows_overlap(out, h0) || rows_overlap(out, lengths) || rows_overlap(h_n, gates) ||
            rows_overlap(h_n, out) || rows_overlap(h_n, lengths) || (p.h_n != p.h0 && rows_overlap(h_n, h0)))
            return set_status(JST_ERR_ARG, "scan: an output overlaps an input");
        return JST_OK;
    }
    if (!p.out_in || !p.dgates) return set_status(JST_ERR_ARG, "scan backward: null out or dgates");
    if (p.ld_dgates < 2 * H || (p.dout && p.ld_dout < H)) return set_status(JST_ERR_ARG, "scan backward: pitch too small");
    if (p.ld_dgates > most || (p.dout && p.ld_dout > most)) return set_status(JST_ERR_ARG, "scan backward: size exceeds 64 bits");
    const ByteRows dgates = matrix(p.dgates, 2 * H, p.ld_dgates), dh0 = vector(p.dh0, state), dh_n = vector(p.dh_n, state);
    for (const ByteRows& in : {gates, matrix(p.out_in, H, p.ld_out), matrix(p.dout, H, p.ld_dout), h0, dh_n, lengths}) {
        if (rows_overlap(dgates, in)) return set_status(JST_ERR_ARG, "scan backward: dgates overlaps an input");
        if (!(in.at == p.dh0 && in.at == p.dh_n) && rows_overlap(dh0, in))
            return set_status(JST_ERR_ARG, "scan backward: dh0 overlaps an input");
    }
    if (rows_overlap(dh0, dgates)) return set_status(JST_ERR_ARG, "scan backward: dh0 overlaps dgates");
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

// For tests: clusters of at most `blocks` blocks, as on a device that places no larger ones.
extern "C" void jst_test_scan_cluster(int blocks) { jst::test_cluster = blocks; }

extern "C" int jst_scan_forward(const float* gates, int64_t ld_gates, int seq, int batch, int hidden, const float* h0,
                                const int32_t* lengths, int reverse, int candidate, float* out, int64_t ld_out,
                                float* h_n, jst_stream_t stream) {
    using namespace jst;
    ScanArgs p{};
    p.gates = gates; p.ld_gates = ld_gates;
    p.h0 = h0; p.lengths = lengths;
    p.out = out; p.ld_out = ld_out; p.h_n = h_n;
    p.seq = seq; p.batch = batch; p.hidden = hidden; p.reverse = reverse != 0;
    int rc = check(p, candidate, false);
    if (rc) return rc;
    rc = require_device();
    if (rc) return rc;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    p.err = device_error_word();
    const int64_t channels = (int64_t)batch * hidden;
    if (channels == 0) return set_status(JST_OK, nullptr);
    if (seq == 0) return pass_state(h_n, h0, channels, s);
    rc = dispatch<false>(p, candidate, s);
    return rc ? rc : launched("scan launch failed");
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
    int rc = check(p, candidate, true);
    if (rc) return rc;
    rc = require_device();
    if (rc) return rc;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    p.err = device_error_word();
    const int64_t channels = (int64_t)batch * hidden;
    if (channels == 0) return set_status(JST_OK, nullptr);
    if (seq == 0) return pass_state(dh0, dh_n, channels, s);
    rc = dispatch<true>(p, candidate, s);
    return rc ? rc : launched("scan backward launch failed");
}
