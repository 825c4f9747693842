// gemm_i8.cu -- the 8-bit integer product on the sm_100a tensor cores
// (tcgen05.mma kind::i8, 32-bit integer accumulators in TMEM, operands staged
// by TMA), for outputs of more than a few rows.
//
//   D[r, s] = sum_k R[r, k] S[s, k]     R: 128 rows a tile, S: BN rows a tile
//
// Both operands are K-major as they are stored, so no pass over them is
// needed.  R are the tokens and S the channels (C[r, s]).
//
// One persistent CTA per SM walks its tiles:
//   warp 0      TMA producer: 128-byte k-slabs (swizzle-128B) into a
//               STAGES-deep ring;
//   warp 1      TMEM allocation and MMA issue into one of two accumulators, so
//               the next tile accumulates while this one is drained;
//   warps 2-9   epilogue, two warps per TMEM lane quadrant on alternate
//               32-column blocks: one scale per lane, one per column (through
//               a 32-entry table in shared memory), bias, ReLU, then a TMA
//               store of the 32 x 32 block (16-byte aligned C), or row by row.
//
// gemm_i8_tokens_kernel: up to 64 tokens, or 64 at a time where tiles are few and
// K is long.  The roles are exchanged (C[s, r]):
// the 128-row side of the instruction holds channels, of which there are
// plenty, and the other the tokens, padded to 16, 32 or 64 instead of 128.  The
// call is a read of the weight, so it has to come from every SM: a cluster of
// CTAs shares a tile's K range and adds its integer sums (exact in any order)
// through distributed shared memory.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <mutex>

#include "gemm_i8.h"
#include "gemm_internal.h"
#include "ptx.cuh"

namespace jst {
namespace i8 {

constexpr int BM = 128;
constexpr int BK = 128;  // int8 elements, one swizzle-128B row
constexpr int THREADS = 320;

template <int BN_, int STAGES_>
struct Cfg {
    static constexpr int BN = BN_;
    static constexpr int STAGES = STAGES_;
    static constexpr uint32_t TMEM_COLS = 2 * BN_;  // two accumulators
    static constexpr uint32_t R_BYTES = BM * BK;
    static constexpr uint32_t S_BYTES = BN_ * BK;
    static constexpr uint32_t STAGE_BYTES = R_BYTES + S_BYTES;
    static constexpr uint32_t STG_OFF = STAGES_ * STAGE_BYTES;  // two 32 x 32 blocks per epilogue warp
    static constexpr uint32_t TAB_OFF = STG_OFF + 8 * 8192;     // a scale and bias table per epilogue warp
    static constexpr uint32_t BAR_OFF = TAB_OFF + 8 * 256;
    static constexpr uint32_t SMEM_BYTES = BAR_OFF + 256 + 768 /*from 256- to 1024-byte alignment*/;
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
    static_assert(S_BYTES % 1024 == 0, "tiles start on swizzle-pattern boundaries");
    static_assert(BN_ >= 32 && TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "TMEM allocation");
    static_assert((2 * STAGES_ + 5) * 8 + 8 <= 256, "barrier area");
};

struct Params {
    int R, S, K;
    int tiles_r, tiles_s;
    float* C;
    int64_t ldc;
    const float* r_scale;
    const float* s_scale;
    const float* bias;  // one per channel
    int relu;
    int tma_store;
    uint32_t* err;
};

// Tile t -> first row of each side: bands of 16 R tiles, so the CTAs of a wave
// share their panels of both operands in L2.
__device__ __forceinline__ void tile_at(int t, const Params& p, int bn, int* r0, int* s0) {
    constexpr int GROUP = 16;
    const int span = GROUP * p.tiles_s;
    const int g = t / span, first = g * GROUP;
    const int gm = min(p.tiles_r - first, GROUP);
    *r0 = (first + (t % span) % gm) * BM;
    *s0 = ((t % span) / gm) * bn;
}

// One epilogue warp's part of a tile: wait for the accumulator at `acc`, drain
// TMEM lane quadrant q's 32-column blocks half, half + 2, ..., release() the
// accumulator after the last read of it, and write C.  The blocks' scales are
// on their way while the accumulator is not complete, and a block is staged
// while the one before it is being stored (STAGED places a warp).  False: a wait gave up.
template <int BN, int STAGED, class Release>
__device__ __forceinline__ bool drain_tile(const Params& p, const CUtensorMap& tm_c, uint32_t acc, uint64_t* complete,
                                           uint32_t phase, volatile uint32_t* err, int r0, int s0, int q, int half,
                                           uint8_t* stage, float* tab, uint32_t& stores, Release release) {
    constexpr int MINE = (BN / 32 + 1) / 2;  // blocks of a warp
    const int lane = threadIdx.x & 31;
    const int row = r0 + q * 32 + lane;
    const float rs = row < p.R ? __ldg(p.r_scale + row) : 0.0f;
    float scale[MINE], bias[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int col = min(s0 + (half + 2 * i) * 32 + lane, p.S - 1);
        scale[i] = __ldg(p.s_scale + col);
        bias[i] = p.bias ? __ldg(p.bias + col) : 0.0f;
    }
    int okw = 0;
    if (lane == 0) okw = ptx::mbar_wait(complete, phase, err) && *err == 0;
    if (!__shfl_sync(0xffffffffu, okw, 0)) return false;
    ptx::tc_fence_after();
    const int nblk = min(BN / 32, (p.S - s0 + 31) / 32);
    const int last = nblk - 1 - ((nblk - 1 - half) & 1);
    if (last < 0) {  // a warp without a block still releases the accumulator
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) release();
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int c = half + 2 * i;
        if (c >= nblk) break;
        const int col0 = s0 + c * 32;
        uint8_t* blk = stage + (stores % STAGED) * 4096;
        uint32_t r[32];
        ptx::tmem_ld_32x32b_x32(acc + ((uint32_t)(q * 32) << 16) + c * 32, r);
        __syncwarp();  // the previous block's readers of the tables are done
        tab[lane] = scale[i];
        tab[32 + lane] = bias[i];
        if (p.tma_store && lane == 0) ptx::bulk_wait_read<STAGED - 1>();  // the store that used `blk` has read it
        ptx::tmem_ld_wait();
        if (c == last) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) release();
        }
        __syncwarp();
        const bool hb = p.bias != nullptr;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 sc = *reinterpret_cast<const float4*>(tab + j);
            const float4 bi = *reinterpret_cast<const float4*>(tab + 32 + j);
            r[j + 0] = __float_as_uint(i8_finish((int)r[j + 0], rs, sc.x, hb, bi.x, p.relu));
            r[j + 1] = __float_as_uint(i8_finish((int)r[j + 1], rs, sc.y, hb, bi.y, p.relu));
            r[j + 2] = __float_as_uint(i8_finish((int)r[j + 2], rs, sc.z, hb, bi.z, p.relu));
            r[j + 3] = __float_as_uint(i8_finish((int)r[j + 3], rs, sc.w, hb, bi.w, p.relu));
        }
        if (p.tma_store) {
            if (r0 + q * 32 < p.R) {  // the box parts past R or S are not written
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *reinterpret_cast<uint4*>(blk + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                        make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    ptx::tma_store_3d(&tm_c, blk, col0, r0 + q * 32, 0);
                    ptx::bulk_commit();
                }
                ++stores;
            }
        } else {  // transpose through shared memory: one 128-byte row segment a store
#pragma unroll
            for (int j = 0; j < 32; ++j)  // word j of row `lane` at j ^ lane: no bank conflicts either way
                reinterpret_cast<uint32_t*>(blk)[lane * 32 + (j ^ lane)] = r[j];
            __syncwarp();
            if (col0 + lane < p.S) {
                float* out = p.C + (int64_t)(r0 + q * 32) * p.ldc + col0 + lane;
                const int rows = min(32, p.R - (r0 + q * 32));
#pragma unroll 8
                for (int j = 0; j < rows; ++j)
                    out[j * p.ldc] = __uint_as_float(reinterpret_cast<uint32_t*>(blk)[j * 32 + (lane ^ j)]);
            }
            ++stores;
        }
    }
    return true;
}

template <class C>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_i8_tc_kernel(const __grid_constant__ CUtensorMap tm_r, const __grid_constant__ CUtensorMap tm_s,
                      const __grid_constant__ CUtensorMap tm_c, const Params p) {
    constexpr int BN = C::BN, STAGES = C::STAGES;
    extern __shared__ __align__(256) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* accf_bar = empty_bar + STAGES;  // [2] accumulator complete (MMA -> epilogue)
    uint64_t* acce_bar = accf_bar + 2;        // [2] accumulator drained (epilogue -> MMA)
    uint64_t* done_bar = acce_bar + 2;        // every MMA of this CTA has completed
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
    volatile uint32_t* err = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int total = p.tiles_r * p.tiles_s;
    const int num_kb = (p.K + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(&accf_bar[b], 1);
            ptx::mbar_init(&acce_bar[b], 8);  // one arrival per epilogue warp
        }
        ptx::mbar_init(done_bar, 1);
        *err = 0;
        ptx::fence_barrier_init();
        ptx::tma_prefetch_desc(&tm_r);
        ptx::tma_prefetch_desc(&tm_s);
        if (p.tma_store) ptx::tma_prefetch_desc(&tm_c);
    }
    if (warp == 1) ptx::tmem_alloc<C::TMEM_COLS>(tmem_slot);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    ptx::griddep_wait();  // may be a programmatic dependent: no global memory before this
    ptx::griddep_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
                int r0, s0;
                tile_at(t, p, BN, &r0, &s0);
                for (int kb = 0; kb < num_kb; ++kb, ++g) {
                    const int s = g % STAGES;
                    if (!ptx::mbar_wait(&empty_bar[s], ((g / STAGES) & 1) ^ 1, err)) {
                        ok = false;
                        break;
                    }
                    uint8_t* st = smem + s * C::STAGE_BYTES;
                    ptx::mbar_arrive_expect_tx(&full_bar[s], C::STAGE_BYTES);
                    ptx::tma_load_3d(st, &tm_r, &full_bar[s], kb * BK, r0, 0);
                    ptx::tma_load_3d(st + C::R_BYTES, &tm_s, &full_bar[s], kb * BK, s0, 0);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = ptx::idesc_i8(BM, BN);
            uint32_t g = 0;
            bool ok = true;
            int i = 0;
            for (int t = blockIdx.x; t < total && ok; t += gridDim.x, ++i) {
                const int buf = i & 1;
                if (!ptx::mbar_wait(&acce_bar[buf], ((i >> 1) & 1) ^ 1, err)) break;
                ptx::tc_fence_after();
                const uint32_t d = tmem_base + buf * BN;
                for (int kb = 0; kb < num_kb; ++kb, ++g) {
                    const int s = g % STAGES;
                    if (!ptx::mbar_wait(&full_bar[s], (g / STAGES) & 1, err)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t st = ptx::smem_u32(smem + s * C::STAGE_BYTES);
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)  // 32 int8 an instruction
                        ptx::mma_i8(d, ptx::smem_desc_kmajor(st + kk * 32, 128),
                                    ptx::smem_desc_kmajor(st + C::R_BYTES + kk * 32, 128), idesc, (kb | kk) != 0);
                    ptx::mma_commit(&empty_bar[s]);
                }
                if (ok) ptx::mma_commit(&accf_bar[buf]);
            }
            ptx::mma_commit(done_bar);  // every MMA completes before the TMEM is released
            ptx::mbar_wait(done_bar, 0, err);
        }
    } else {
        const int q = warp & 3;            // TMEM lane quadrant this warp may access
        const int half = (warp - 2) >> 2;  // 0: even 32-column blocks, 1: odd
        uint8_t* blk = smem + C::STG_OFF + (warp - 2) * 8192;
        float* tab = reinterpret_cast<float*>(smem + C::TAB_OFF + (warp - 2) * 256);  // [32] scale, [32] bias
        uint32_t stores = 0;  // blocks staged by this warp
        int i = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x, ++i) {
            const int buf = i & 1;
            int r0, s0;
            tile_at(t, p, BN, &r0, &s0);
            if (!drain_tile<BN, 2>(p, tm_c, tmem_base + buf * BN, &accf_bar[buf], (i >> 1) & 1, err, r0, s0, q, half,
                                blk, tab, stores, [&] { ptx::mbar_arrive(&acce_bar[buf]); }))
                break;
        }
        if (lane == 0 && stores) ptx::bulk_wait_all();  // C is written before the CTA exits
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        ptx::tc_fence_after();
        ptx::tmem_dealloc<C::TMEM_COLS>(tmem_base);
    }
    if (threadIdx.x == 0 && *err != 0) atomicOr(p.err, *err);
}

// ------------------------------------------------------------ pairs of SMs
// The same walk with 256 x 256 tiles on two CTAs of a cluster (cta_group::2):
// each stages its 128 rows of R and of S, each half of S serves both, and one
// thread of the first issues the instructions for the two.  A CTA alone reads
// and writes 192 bytes of shared memory for what takes the pair 128 a CTA, and
// shared memory is what bounds gemm_i8_tc_kernel (128 bytes a cycle).
// Barriers of the first CTA count both CTAs' loads and drained accumulators;
// commits arrive at both.
struct PairCfg {
    static constexpr int STAGES = 6;
    static constexpr int BN = 256;
    static constexpr uint32_t HALF_BYTES = BM * BK;  // 128 rows of R, 128 rows of S
    static constexpr uint32_t STAGE_BYTES = 2 * HALF_BYTES;
    static constexpr uint32_t STG_OFF = STAGES * STAGE_BYTES;
    static constexpr uint32_t TAB_OFF = STG_OFF + 8 * 4096;  // one 32 x 32 block a warp: a sixth stage is worth more (8192^3: 365 us; five and two blocks 384)
    static constexpr uint32_t BAR_OFF = TAB_OFF + 8 * 256;
    static constexpr uint32_t SMEM_BYTES = BAR_OFF + 256 + 768;
    static_assert(SMEM_BYTES <= 227 * 1024 && (2 * STAGES + 5) * 8 + 8 <= 256, "shared memory per CTA");
};

__device__ __forceinline__ void pair_tile_at(int t, const Params& p, int* r0, int* s0) {
    constexpr int GROUP = 8;  // bands of 8 x 256 rows
    const int span = GROUP * p.tiles_s;
    const int g = t / span, first = g * GROUP;
    const int gm = min(p.tiles_r - first, GROUP);
    *r0 = (first + (t % span) % gm) * 2 * BM;
    *s0 = ((t % span) / gm) * PairCfg::BN;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tm_r, const __grid_constant__ CUtensorMap tm_s,
                        const __grid_constant__ CUtensorMap tm_c, const Params p) {
    using C = PairCfg;
    constexpr int STAGES = C::STAGES;
    extern __shared__ __align__(256) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);  // of the first CTA: both halves have landed
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* accf_bar = empty_bar + STAGES;  // [2]
    uint64_t* acce_bar = accf_bar + 2;        // [2] of the first CTA: both CTAs have drained it
    uint64_t* done_bar = acce_bar + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
    volatile uint32_t* err = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x & 1);
    const int pairs = (int)(gridDim.x >> 1), pair = (int)(blockIdx.x >> 1);
    const int total = p.tiles_r * p.tiles_s;
    const int num_kb = (p.K + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(&accf_bar[b], 1);
            ptx::mbar_init(&acce_bar[b], 16);  // one arrival per epilogue warp of either CTA
        }
        ptx::mbar_init(done_bar, 1);
        *err = 0;
        ptx::fence_barrier_init();
        ptx::tma_prefetch_desc(&tm_r);
        ptx::tma_prefetch_desc(&tm_s);
        if (p.tma_store) ptx::tma_prefetch_desc(&tm_c);
    }
    if (warp == 1) ptx::tmem_alloc_pair<512>(tmem_slot);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_arrive();  // the other CTA's barriers and TMEM are ready too
    ptx::cluster_wait();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            bool ok = true;
            for (int t = pair; t < total && ok; t += pairs) {
                int r0, s0;
                pair_tile_at(t, p, &r0, &s0);
                for (int kb = 0; kb < num_kb; ++kb, ++g) {
                    const int s = g % STAGES;
                    if (!ptx::mbar_wait(&empty_bar[s], ((g / STAGES) & 1) ^ 1, err)) {
                        ok = false;
                        break;
                    }
                    uint8_t* st = smem + s * C::STAGE_BYTES;
                    const uint32_t bar = ptx::cluster_addr(ptx::smem_u32(&full_bar[s]), 0);
                    if (rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
                    ptx::tma_load_3d_pair(st, &tm_r, bar, kb * BK, r0 + rank * BM, 0);
                    ptx::tma_load_3d_pair(st + C::HALF_BYTES, &tm_s, bar, kb * BK, s0 + rank * BM, 0);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = ptx::idesc_i8(2 * BM, C::BN);
            uint32_t g = 0;
            bool ok = true;
            int i = 0;
            for (int t = pair; t < total && ok; t += pairs, ++i) {
                const int buf = i & 1;
                if (!ptx::mbar_wait<true>(&acce_bar[buf], ((i >> 1) & 1) ^ 1, err)) break;
                ptx::tc_fence_after();
                const uint32_t d = tmem_base + buf * C::BN;
                for (int kb = 0; kb < num_kb; ++kb, ++g) {
                    const int s = g % STAGES;
                    if (!ptx::mbar_wait(&full_bar[s], (g / STAGES) & 1, err)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after();
                    const uint32_t st = ptx::smem_u32(smem + s * C::STAGE_BYTES);
#pragma unroll
                    for (int kk = 0; kk < BK / 32; ++kk)
                        ptx::mma_i8_pair(d, ptx::smem_desc_kmajor(st + kk * 32, 128),
                                         ptx::smem_desc_kmajor(st + C::HALF_BYTES + kk * 32, 128), idesc, (kb | kk) != 0);
                    ptx::mma_commit_pair(&empty_bar[s]);
                }
                if (ok) ptx::mma_commit_pair(&accf_bar[buf]);
            }
            ptx::mma_commit_pair(done_bar);
            ptx::mbar_wait(done_bar, 0, err);  // every MMA completes before the TMEM is released
        }
        __syncwarp();
    } else {
        const int q = warp & 3;
        const int half = (warp - 2) >> 2;
        uint8_t* blk = smem + C::STG_OFF + (warp - 2) * 4096;
        float* tab = reinterpret_cast<float*>(smem + C::TAB_OFF + (warp - 2) * 256);
        uint32_t stores = 0;  // blocks staged by this warp
        int i = 0;
        for (int t = pair; t < total; t += pairs, ++i) {
            const int buf = i & 1;
            int r0, s0;
            pair_tile_at(t, p, &r0, &s0);
            r0 += rank * BM;
            const uint32_t drained = ptx::cluster_addr(ptx::smem_u32(&acce_bar[buf]), 0);
            if (!drain_tile<C::BN, 1>(p, tm_c, tmem_base + buf * C::BN, &accf_bar[buf], (i >> 1) & 1, err, r0, s0, q, half,
                                   blk, tab, stores, [&] { ptx::mbar_arrive_cluster(drained); }))
                break;
        }
        if (lane == 0 && stores) ptx::bulk_wait_all();
        __syncwarp();
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == 0) {  // the last commit's arrival here, before this CTA may leave
        if (lane == 0 && rank == 1) ptx::mbar_wait(done_bar, 0, err);
        __syncwarp();
    }
    ptx::cluster_arrive();  // neither CTA leaves, or frees its TMEM, while the other's work may touch it
    ptx::cluster_wait();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair<512>(tmem_base);
    }
    if (threadIdx.x == 0 && *err != 0) atomicOr(p.err, *err);
}

// ------------------------------------------------------------ few tokens
// FP32: the tokens come as fp32 rows.  Every CTA finds their scales and
// quantises its own part of K into shared memory while its weight is on the way.
template <int T_, int STAGES_, bool FP32_ = false>
struct TokCfg {
    static constexpr int T = T_;  // tokens, padded
    static constexpr int STAGES = STAGES_;
    static constexpr bool FP32 = FP32_;
    static constexpr int SLABS = 16;  // FP32: k-slabs of a CTA at most
    static constexpr uint32_t TMEM_COLS = T_ < 32 ? 32 : T_;
    static constexpr uint32_t R_BYTES = BM * BK;
    static constexpr uint32_t S_BYTES = T_ * BK;
    static constexpr uint32_t STAGE_BYTES = R_BYTES + (FP32_ ? 0 : S_BYTES);
    static constexpr uint32_t X_OFF = STAGES_ * STAGE_BYTES;  // FP32: [SLABS] tiles of the tokens
    static constexpr uint32_t EX_OFF = X_OFF + (FP32_ ? SLABS * S_BYTES : 0);  // int32 [cluster][128][tokens of this CTA]
    static constexpr uint32_t SCALE_OFF = EX_OFF + T_ * BM * 4;
    static constexpr uint32_t BAR_OFF = SCALE_OFF + 256;
    static constexpr uint32_t SMEM_BYTES = BAR_OFF + 256 + 768 /*from 256- to 1024-byte alignment*/;
    static_assert(SMEM_BYTES <= 227 * 1024 && S_BYTES % 1024 == 0 && (2 * STAGES_ + 2) * 8 + 8 <= 256, "shared memory");
};
constexpr int TOK_THREADS = 192;

struct TokParams {
    int channels, tokens, K;
    int cluster_log2, kb_per_rank;  // CTAs that share a tile (at most T / 4), k-slabs of each
    float* C;
    int64_t ldc;
    const float* channel_scale;
    const float* token_scale;
    const float* bias;
    int relu;
    uint32_t* err;
    const float* x;  // FP32: the tokens
    int64_t ldx;
};

// FP32: warp w of four takes tokens w, w + 4, ...: the scale of the whole row,
// then the row's part of K as the swizzled tiles that TMA would have written
// (16-byte piece j of a 128-byte row r at j ^ (r & 7)), zeros behind M and K.
template <class C>
__device__ __forceinline__ void quantize_tokens(const TokParams& p, uint8_t* smem, float* token_scale, uint64_t* x_bar,
                                                int kb0, int num_kb, int own0, int own, int w, int lane) {
    constexpr int ROWS = C::T / 4;  // of a warp, side by side: their loads are in flight together
    const bool vec = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && (p.tokens == 1 || (p.ldx & 3) == 0);
    auto fetch = [&](int m, int k) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float* at = p.x + (int64_t)m * p.ldx + k;
        if (m >= p.tokens) return v;
        if (vec && k + 4 <= p.K) return __ldg(reinterpret_cast<const float4*>(at));
        if (k < p.K) v.x = __ldg(at);
        if (k + 1 < p.K) v.y = __ldg(at + 1);
        if (k + 2 < p.K) v.z = __ldg(at + 2);
        if (k + 3 < p.K) v.w = __ldg(at + 3);
        return v;
    };
    uint32_t peak[ROWS] = {};
#pragma unroll 2
    for (int k = 4 * lane; k < p.K; k += 128) {
        float4 v[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) v[i] = fetch(w + 4 * i, k);
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
            peak[i] = max(max(max(peak[i], abs_bits(v[i].x)), max(abs_bits(v[i].y), abs_bits(v[i].z))), abs_bits(v[i].w));
    }
    // A lane a row: the divisions of all rows at once (5 x 2048 x 512: one row after the other, 0.4 us more).
    uint32_t of_mine = 0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const uint32_t of_row = __reduce_max_sync(0xffffffffu, peak[i]);
        if (lane == i) of_mine = of_row;
    }
    const float my_scale = row_scale(of_mine), my_inverse = row_inverse(my_scale);
    const int my_row = w + 4 * lane - own0;
    if (lane < ROWS && my_row >= 0 && my_row < own) token_scale[my_row] = my_scale;
    float s[ROWS], inv[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        s[i] = __shfl_sync(0xffffffffu, my_scale, i);
        inv[i] = __shfl_sync(0xffffffffu, my_inverse, i);
    }
#pragma unroll 2
    for (int kb = 0; kb < num_kb; ++kb) {
        float4 v[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) v[i] = fetch(w + 4 * i, (kb0 + kb) * BK + 4 * lane);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const int m = w + 4 * i;
            uint8_t* tile = smem + C::X_OFF + kb * C::S_BYTES + m * BK;
            *reinterpret_cast<uint32_t*>(tile + (((lane >> 2) ^ (m & 7)) << 4) + ((lane & 3) << 2)) = quantize4(v[i], s[i], inv[i]);
        }
    }
    ptx::fence_proxy_async_smem();  // the tensor cores read what these stores wrote
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(x_bar);
}

//   warp 0      TMA producer (and, before it may read what the launch before
//               this one wrote, prefetches of its weight slabs into L2)
//   warp 1      TMEM allocation, MMA issue
//   warps 2-5   exchange and epilogue, a lane a channel
template <class C>
__global__ void __launch_bounds__(TOK_THREADS)
    gemm_i8_tokens_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                          const TokParams p) {
    constexpr int STAGES = C::STAGES;
    extern __shared__ __align__(256) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int* exchange = reinterpret_cast<int*>(smem + C::EX_OFF);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
    uint64_t* empty_bar = full_bar + STAGES;
    uint64_t* accum_bar = empty_bar + STAGES;
    uint64_t* x_bar = accum_bar + 1;  // FP32: the tokens are quantised
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(x_bar + 1);
    volatile uint32_t* err = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* token_scale = reinterpret_cast<float*>(smem + C::SCALE_OFF);
    const int cluster = 1 << p.cluster_log2;
    const int rank = (int)(blockIdx.x & (cluster - 1));
    const int n0 = (int)(blockIdx.x >> p.cluster_log2) * BM;
    const int kb0 = rank * p.kb_per_rank;
    const int num_kb = max(0, min((p.K + BK - 1) / BK - kb0, p.kb_per_rank));
    const int own = C::T >> p.cluster_log2, own0 = rank * own;  // the tokens whose sums meet in this CTA: a multiple of 4
    const int m0 = blockIdx.y * C::T, tokens = p.tokens - m0;   // FP32: m0 is 0

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full_bar[s], 1);
            ptx::mbar_init(&empty_bar[s], 1);
        }
        ptx::mbar_init(accum_bar, 1);
        ptx::mbar_init(x_bar, 4);  // one arrival per quantising warp
        *err = 0;
        ptx::fence_barrier_init();
        ptx::tma_prefetch_desc(&tm_w);
        if (!C::FP32) ptx::tma_prefetch_desc(&tm_x);
        // no more of a long row than fits L2 for all CTAs together
        for (int kb = 0; kb < min(num_kb, 16); ++kb) ptx::tma_prefetch_3d(&tm_w, (kb0 + kb) * BK, n0, 0);
    }
    if (warp == 1) ptx::tmem_alloc<C::TMEM_COLS>(tmem_slot);
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    ptx::griddep_wait();
    ptx::griddep_launch_dependents();
    if (!C::FP32 && threadIdx.x < own) 
        token_scale[threadIdx.x] = own0 + (int)threadIdx.x < tokens ? __ldg(p.token_scale + m0 + own0 + threadIdx.x) : 0.0f;
    if (cluster > 1) {  // nobody writes another's shared memory before that one runs
        ptx::cluster_arrive();
        ptx::cluster_wait();
    }

    if (warp == 0) {
        if (lane == 0) {
            for (int kb = 0; kb < num_kb; ++kb) {
                const int s = kb % STAGES;
                if (!ptx::mbar_wait(&empty_bar[s], ((kb / STAGES) & 1) ^ 1, err)) break;
                uint8_t* st = smem + s * C::STAGE_BYTES;
                ptx::mbar_arrive_expect_tx(&full_bar[s], C::STAGE_BYTES);
                ptx::tma_load_3d(st, &tm_w, &full_bar[s], (kb0 + kb) * BK, n0, 0);
                if (!C::FP32) ptx::tma_load_3d(st + C::R_BYTES, &tm_x, &full_bar[s], (kb0 + kb) * BK, m0, 0);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = ptx::idesc_i8(BM, C::T);
            const bool ready = !C::FP32 || ptx::mbar_wait(x_bar, 0, err);
            for (int kb = 0; kb < num_kb && ready; ++kb) {
                const int s = kb % STAGES;
                if (!ptx::mbar_wait(&full_bar[s], (kb / STAGES) & 1, err)) break;
                ptx::tc_fence_after();
                const uint32_t st = ptx::smem_u32(smem + s * C::STAGE_BYTES);
                const uint32_t xt = C::FP32 ? ptx::smem_u32(smem + C::X_OFF + kb * C::S_BYTES) : st + C::R_BYTES;
#pragma unroll
                for (int kk = 0; kk < BK / 32; ++kk)
                    ptx::mma_i8(tmem_base, ptx::smem_desc_kmajor(st + kk * 32, 128),
                                ptx::smem_desc_kmajor(xt + kk * 32, 128), idesc, (kb | kk) != 0);
                ptx::mma_commit(&empty_bar[s]);
            }
            ptx::mma_commit(accum_bar);  // always signalled, also on the error path
            ptx::mbar_wait(accum_bar, 0, err);
        }
        __syncwarp();
    } else {
        if (C::FP32) quantize_tokens<C>(p, smem, token_scale, x_bar, kb0, num_kb, own0, own, warp - 2, lane);
        int okw = 0;
        if (lane == 0) okw = ptx::mbar_wait(accum_bar, 0, err) && *err == 0;
        const bool ok = __shfl_sync(0xffffffffu, okw, 0) != 0;
        ptx::tc_fence_after();
        const int q = warp & 3;  // TMEM lane quadrant this warp may access
        const int row = q * 32 + lane;
        if (ok) {
            // this lane's channel: its partial sums of the tokens, four at a
            // time, to the CTA that owns those
#pragma unroll 1
            for (int c = 0; c < C::T && c < tokens; c += 16) {
                uint32_t r[16];
                if (num_kb > 0) {
                    ptx::tmem_ld_32x32b_x16(tmem_base + ((uint32_t)(q * 32) << 16) + c, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) r[j] = 0;
                }
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const int owner = (c + j) / own, at = (rank * BM + row) * own + (c + j) % own;  // own: a power of two
                    if (cluster > 1)
                        ptx::cluster_store_v4(ptx::cluster_addr(ptx::smem_u32(exchange + at), owner), r[j], r[j + 1],
                                              r[j + 2], r[j + 3]);
                    else
                        *reinterpret_cast<uint4*>(exchange + at) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                }
            }
        }
    }
    ptx::tc_fence_before();
    if (cluster > 1) {  // every sum has arrived; nobody leaves before
        ptx::cluster_arrive();
        ptx::cluster_wait();
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<C::TMEM_COLS>(tmem_base);
    } else if (warp >= 2 && *err == 0) {
        const int row = (warp & 3) * 32 + lane, n = n0 + row;
        if (n < p.channels) {
            const float cs = __ldg(p.channel_scale + n), bias = p.bias ? __ldg(p.bias + n) : 0.0f;
            float* out = p.C + (int64_t)(m0 + own0) * p.ldc + n;
            for (int i = 0; i < own && own0 + i < tokens; i += 4) {
                int4 sum = make_int4(0, 0, 0, 0);
                for (int o = 0; o < cluster; ++o) {
                    const int4 v = *reinterpret_cast<const int4*>(exchange + (o * BM + row) * own + i);
                    sum = make_int4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
                }
                const int v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (own0 + i + j < tokens)
                        out[(i + j) * p.ldc] = i8_finish(v[j], token_scale[i + j], cs, p.bias != nullptr, bias, p.relu);
            }
        }
    }
    if (threadIdx.x == 0 && *err != 0) atomicOr(p.err, *err);
}

// Rows without 16-byte alignment -> rows of pitch ldd in a workspace.
__global__ void realign_rows_kernel(const int8_t* __restrict__ src, int64_t lds, int rows, int cols,
                                    int8_t* __restrict__ dst, int64_t ldd) {
    ptx::griddep_wait();
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (int k = 4 * threadIdx.x; k < cols; k += 4 * blockDim.x) {
            const int8_t* s = src + r * lds + k;
            uint32_t v = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (k + j < cols) v |= (uint32_t)(uint8_t)s[j] << (8 * j);
            *reinterpret_cast<uint32_t*>(dst + r * ldd + k) = v;  // ldd is a multiple of 16: the pad is this row's own
        }
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// rows x inner elements of elem_bytes each, `pitch` elements apart; box: one
// 128-byte row of box_rows rows, swizzle-128B.
static bool make_map(CUtensorMap* m, const void* base, CUtensorMapDataType type, int elem_bytes, int64_t inner,
                     int64_t rows, int64_t pitch, int box_rows) {
    auto enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, 1};
    const cuuint64_t strides[2] = {(cuuint64_t)(pitch * elem_bytes), (cuuint64_t)(pitch * elem_bytes * rows)};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / elem_bytes), (cuuint32_t)box_rows, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    return enc(m, type, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class Cf>
static int launch(const CUtensorMap& r, const CUtensorMap& s, const CUtensorMap& c, const Params& p, cudaStream_t st) {
    static bool attr_set[64] = {};
    static std::mutex mu;
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 0 && dev < 64 && !attr_set[dev]) {
            if (cudaFuncSetAttribute(gemm_i8_tc_kernel<Cf>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     Cf::SMEM_BYTES) != cudaSuccess)
                return set_status(JST_ERR_CUDA, "cudaFuncSetAttribute(gemm_i8_tc_kernel) failed");
            attr_set[dev] = true;
        }
    }
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)p.tiles_r * p.tiles_s, sm_count());
    ProfScope prof(st, KID_GEMM_I8);
    if (launch_dependent(gemm_i8_tc_kernel<Cf>, dim3(grid), dim3(THREADS), Cf::SMEM_BYTES, st, r, s, c, p) !=
        cudaSuccess)
        return set_status(JST_ERR_CUDA, "gemm_i8_tc_kernel launch failed");
    return JST_OK;
}

static bool aligned(const int8_t* x, int64_t ld, int rows) {
    return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (rows == 1 || (ld & 15) == 0);
}

static int realign(const int8_t** x, int64_t* ld, int rows, int cols, int8_t* to, cudaStream_t s) {
    const int64_t ldd = ((int64_t)cols + 15) / 16 * 16;
    {
        ProfScope prof(s, KID_QUANT);
        if (launch_dependent(realign_rows_kernel, dim3((unsigned)std::min(rows, 148 * 16)), dim3(128), 0, s, *x, *ld,
                             rows, cols, to, ldd) != cudaSuccess)
            return set_status(JST_ERR_CUDA, "realign_rows launch failed");
    }
    *x = to;
    *ld = ldd;
    return JST_OK;
}

static int launch_pair(const CUtensorMap& r, const CUtensorMap& s, const CUtensorMap& c, const Params& p, cudaStream_t st) {
    static bool attr_set[64] = {};
    static std::mutex mu;
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 0 && dev < 64 && !attr_set[dev]) {
            if (cudaFuncSetAttribute(gemm_i8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     PairCfg::SMEM_BYTES) != cudaSuccess)
                return set_status(JST_ERR_CUDA, "cudaFuncSetAttribute(gemm_i8_pair_kernel) failed");
            attr_set[dev] = true;
        }
    }
    const unsigned grid = 2 * (unsigned)std::min<int64_t>((int64_t)p.tiles_r * p.tiles_s, sm_count() / 2);
    ProfScope prof(st, KID_GEMM_I8);
    if (launch_dependent(gemm_i8_pair_kernel, dim3(grid), dim3(THREADS), PairCfg::SMEM_BYTES, st, r, s, c, p) != cudaSuccess)
        return set_status(JST_ERR_CUDA, "gemm_i8_pair_kernel launch failed");
    return JST_OK;
}

template <class Cf>
static int launch_tokens(const CUtensorMap& w, const CUtensorMap& x, const TokParams& p, cudaStream_t st) {
    static bool attr_set[64] = {};
    static std::mutex mu;
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 0 && dev < 64 && !attr_set[dev]) {
            if (cudaFuncSetAttribute(gemm_i8_tokens_kernel<Cf>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     Cf::SMEM_BYTES) != cudaSuccess)
                return set_status(JST_ERR_CUDA, "cudaFuncSetAttribute(gemm_i8_tokens_kernel) failed");
            attr_set[dev] = true;
        }
    }
    const int cluster = 1 << p.cluster_log2;
    const dim3 grid((unsigned)((p.channels + BM - 1) / BM * cluster), (unsigned)((p.tokens + Cf::T - 1) / Cf::T));
    ProfScope prof(st, KID_GEMM_I8);
    if (launch_dependent_cluster(gemm_i8_tokens_kernel<Cf>, grid, dim3(TOK_THREADS), cluster, Cf::SMEM_BYTES, st,
                                 w, x, p) != cudaSuccess)
        return set_status(JST_ERR_CUDA, "gemm_i8_tokens_kernel launch failed");
    return JST_OK;
}

// The pitch of a single row is never used, but a map wants a multiple of 16 bytes.
static bool make_operand_map(CUtensorMap* m, const int8_t* x, int rows, int K, int64_t ld, int box_rows) {
    return make_map(m, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K, rows, rows == 1 ? ((int64_t)K + 15) / 16 * 16 : ld, box_rows);
}

static int64_t tokens_tiles(const I8Args& a, int T) { return (int64_t)((a.N + BM - 1) / BM) * ((a.M + T - 1) / T); }

// CTAs that share a tile of T tokens: as many as the SMs take (two CTAs of up to
// 32 tokens fit one), with a k-slab and four tokens at least each (16 tokens,
// 4096 x 4096: 15.6 us alone, 10.4 with two, 7.9 with four; 16, 2048 x 512:
// 5.3, 4.8, 4.2; 64, 8192 x 8192: 34.1, 21.6, and 28.4 with four, which no
// longer run at the same time).  A cluster keeps to one GPC, so the last SMs of
// each stay empty: of clusters of 4, 33 run at once and 34 do not (64, 4224 x 4096
// 11.1 us, 4352 x 4096 18.7, with two 14.1), of 8, 15 and not 16 (1920 x 4096 9.1,
// 2048 x 4096 15.6, with four 9.6).
static int tokens_cluster_log2(const I8Args& a, int T) {
    const int64_t tiles = tokens_tiles(a, T);
    const int slabs = (a.K + BK - 1) / BK, room = sm_count() * (T <= 32 ? 2 : 1), percent[] = {100, 88, 80};
    int lg = 0;
    while (lg < 3 && (8 << lg) <= T && (tiles << (lg + 1)) <= room * percent[lg] / 100 && (2 << lg) <= slabs) ++lg;
    return lg;
}

// x: the tokens in fp32 (gemm_i8_tc_takes_fp32), or null.
static int run_tokens(const I8Args& a, const float* x, int64_t ldx, cudaStream_t s) {
    const int T = a.M <= 16 ? 16 : a.M <= 32 ? 32 : 64;
    CUtensorMap w, xm;
    if (!make_operand_map(&w, a.B, a.N, a.K, a.ldb, BM)) return set_status(JST_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    xm = w;  // not read with fp32 tokens
    if (!x && !make_operand_map(&xm, a.A, a.M, a.K, a.lda, T)) return set_status(JST_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    TokParams p{};
    p.channels = a.N; p.tokens = a.M; p.K = a.K;
    p.C = a.C; p.ldc = a.ldc;
    p.channel_scale = a.b_scale; p.token_scale = a.a_scale;
    p.bias = a.bias; p.relu = a.relu;
    p.err = device_error_word();
    const int lg = tokens_cluster_log2(a, T), slabs = (a.K + BK - 1) / BK;
    p.cluster_log2 = lg;
    p.kb_per_rank = (slabs + (1 << lg) - 1) >> lg;
    p.x = x;
    p.ldx = ldx;
    if (x) return launch_tokens<TokCfg<16, 4, true>>(w, xm, p, s);
    if (T == 16) return launch_tokens<TokCfg<16, 5>>(w, xm, p, s);
    if (T == 32) return launch_tokens<TokCfg<32, 4>>(w, xm, p, s);
    return launch_tokens<TokCfg<64, 7>>(w, xm, p, s);
}

static int run_aligned(const I8Args& a, cudaStream_t s) {
    if (a.M <= 64) return run_tokens(a, nullptr, 0, s);
    // The tile by what it is expected to take, in ns measured on a B200: a k-slab
    // (8192^3: 365 us in pairs, 602 and 1055 in tiles of 128 and 64 columns) or,
    // where K is short, the epilogue (8192 x 8192 x 512: 93, 66, 93) of a tile,
    // times the waves of tiles, and one of each at the ends.  (256 x 8192 x 8192:
    // 31.5, 25.1, 42.1; 128 x 8192 x 8192: 39.9, 25.1, 23.4; 2048^3: 19.4, 16.4,
    // 23.9; 3000^3: 25.8, 36.2, 62.8.)
    const struct { int rows, cols, slots, slab_ns, epilogue_ns; } kinds[] = {
        {2 * BM, 256, sm_count() / 2, 410, 6500}, {BM, 128, sm_count(), 336, 2400}, {BM, 64, sm_count(), 294, 1650}};
    int bn = 0;
    int64_t best = INT64_MAX;
    for (const auto& k : kinds) {
        const int64_t tiles = (int64_t)((a.M + k.rows - 1) / k.rows) * ((a.N + k.cols - 1) / k.cols);
        const int64_t waves = (tiles + k.slots - 1) / k.slots, slabs = (int64_t)((a.K + BK - 1) / BK) * k.slab_ns;
        const int64_t cost = (waves - 1) * std::max<int64_t>(slabs, k.epilogue_ns) + slabs + k.epilogue_ns;
        if (cost < best) {
            best = cost;
            bn = k.cols;
        }
    }
    // Few tiles and a long K: the kernel of few tokens, 64 at a time, whose clusters
    // share K, at 350 ns a k-slab and an exchange that shrinks with a CTA's part of
    // the tile (us: 200 x 300 x 8192 takes 10.0, in tiles 22.1, 200 x 1024 x 4096 10.2 and
    // 13.0; 1000 x 1024 x 8192 would take 29.0, in tiles 22.9).
    const int lg = tokens_cluster_log2(a, 64), slabs = (a.K + BK - 1) / BK;
    const int exchange_ns[] = {7650, 6350, 5950, 4450};
    if (lg > 0 && exchange_ns[lg] + (int64_t)((slabs + (1 << lg) - 1) >> lg) * 350 < best) return run_tokens(a, nullptr, 0, s);
    const bool pair = bn == 256;
    Params p{};
    p.R = a.M; p.S = a.N; p.K = a.K;
    p.C = a.C; p.ldc = a.ldc;
    p.r_scale = a.a_scale; p.s_scale = a.b_scale;
    p.bias = a.bias; p.relu = a.relu;
    p.err = device_error_word();
    p.tiles_r = pair ? (p.R + 2 * BM - 1) / (2 * BM) : (p.R + BM - 1) / BM;
    p.tiles_s = (p.S + bn - 1) / bn;
    if ((int64_t)p.tiles_r * p.tiles_s > 0x7fffffff) return set_status(JST_ERR_ARG, "gemm_i8: too many tiles");
    CUtensorMap mr, ms, mc;
    if (!make_operand_map(&mr, a.A, a.M, a.K, a.lda, BM) || !make_operand_map(&ms, a.B, a.N, a.K, a.ldb, pair ? BM : bn))
        return set_status(JST_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    mc = mr;  // not read unless tma_store
    p.tma_store = (reinterpret_cast<uintptr_t>(a.C) & 15) == 0 && (a.ldc & 3) == 0 &&
                  make_map(&mc, a.C, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, a.N, a.M, a.ldc, 32);
    if (pair) return launch_pair(mr, ms, mc, p, s);
    if (bn == 128) return launch<Cfg<128, 5>>(mr, ms, mc, p, s);
    return launch<Cfg<64, 6>>(mr, ms, mc, p, s);
}

}  // namespace i8

// Up to 16 tokens of so few values that one launch beats two: such calls wait
// for the host, which spends 4.4 us on this one and 7.5 on a quantisation, its
// workspace and the product (5 x 2048 x 512: a call takes 5.5 and 9.3 us, and on the
// device alone 6.2 and 5.5; 2 x 4096 x 1024, 7.2 and 9.5, 7.8 and 5.9).  The weight needs no copy.
bool gemm_i8_tc_takes_fp32(const I8Args& a) {
    return a.M <= 16 && (int64_t)a.M * a.K <= 4096 && a.K <= i8::TokCfg<16, 4, true>::SLABS * i8::BK &&
           i8::aligned(a.B, a.ldb, a.N);
}

int gemm_i8_tc_run_fp32(const I8Args& a, const float* x, int64_t ldx, cudaStream_t s) {
    return i8::run_tokens(a, x, ldx, s);
}

bool gemm_i8_tc_in_place(const I8Args& a) {
    return i8::aligned(a.A, a.lda, a.M) && i8::aligned(a.B, a.ldb, a.N);
}

int gemm_i8_tc_run(const I8Args& args, cudaStream_t s) {
    I8Args a = args;
    const bool copy_a = !i8::aligned(a.A, a.lda, a.M), copy_b = !i8::aligned(a.B, a.ldb, a.N);
    const size_t pitch = ((size_t)a.K + 15) / 16 * 16;
    void* ws = nullptr;
    if (copy_a || copy_b) {
        const int rc = workspace_alloc(pitch * ((copy_a ? (size_t)a.M : 0) + (copy_b ? (size_t)a.N : 0)), s, &ws);
        if (rc) return rc;
    }
    int8_t* to = static_cast<int8_t*>(ws);
    int rc = copy_a ? i8::realign(&a.A, &a.lda, a.M, a.K, to, s) : JST_OK;
    if (!rc && copy_b) rc = i8::realign(&a.B, &a.ldb, a.N, a.K, to + (copy_a ? pitch * a.M : 0), s);
    if (!rc) rc = i8::run_aligned(a, s);
    const int frc = ws ? workspace_free(ws, s) : JST_OK;
    return rc ? rc : frc;
}

}  // namespace jst
