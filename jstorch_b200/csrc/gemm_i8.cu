// gemm_i8.cu -- the 8-bit integer product on the sm_100a tensor cores
// (tcgen05.mma kind::i8, 32-bit integer accumulators in TMEM, operands staged
// by TMA), for outputs of more than a few rows.
//
//   D[r, s] = sum_k R[r, k] S[s, k]     R: 128 rows a tile, S: BN rows a tile
//
// Both operands are K-major as they are stored, so no pass over them is
// needed.  With many tokens R are the tokens and S the channels (C[r, s]).
// With few tokens the roles are exchanged (SWAP, C[s, r]): the 128-row side
// of the instruction then holds channels, of which there are plenty, and the
// BN side holds the tokens, padded to 16, 32 or 64 instead of 128.
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
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
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
    static constexpr uint32_t ACC_COLS = BN_ < 32 ? 32 : BN_;  // the epilogue reads 32 columns at a time
    static constexpr uint32_t TMEM_COLS = 2 * ACC_COLS;
    static constexpr uint32_t R_BYTES = BM * BK;
    static constexpr uint32_t S_BYTES = BN_ * BK;
    static constexpr uint32_t STAGE_BYTES = R_BYTES + S_BYTES;
    static constexpr uint32_t STG_OFF = STAGES_ * STAGE_BYTES;  // a 32 x 32 block per epilogue warp
    static constexpr uint32_t TAB_OFF = STG_OFF + 8 * 4096;     // a scale and bias table per epilogue warp
    static constexpr uint32_t BAR_OFF = TAB_OFF + 8 * 256;
    static constexpr uint32_t SMEM_BYTES = BAR_OFF + 256 + 768 /*from 256- to 1024-byte alignment*/;
    static_assert(SMEM_BYTES <= 227 * 1024, "shared memory per CTA");
    static_assert(S_BYTES % 1024 == 0, "tiles start on swizzle-pattern boundaries");
    static_assert(TMEM_COLS >= 32 && TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "TMEM allocation");
    static_assert((2 * STAGES_ + 5) * 8 + 8 <= 256, "barrier area");
};

struct Params {
    int R, S, K;
    int tiles_r, tiles_s;
    float* C;
    int64_t ldc;
    const float* r_scale;
    const float* s_scale;
    const float* bias;  // one per channel: of S, or of R when swapped
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

template <class C, bool SWAP>
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
                const uint32_t d = tmem_base + buf * C::ACC_COLS;
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
        uint8_t* blk = smem + C::STG_OFF + (warp - 2) * 4096;
        float* tab = reinterpret_cast<float*>(smem + C::TAB_OFF + (warp - 2) * 256);  // [32] scale, [32] bias
        bool stored = false;
        int i = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x, ++i) {
            const int buf = i & 1;
            int r0, s0;
            tile_at(t, p, BN, &r0, &s0);
            const int row = r0 + q * 32 + lane;
            const float rs = row < p.R ? __ldg(p.r_scale + row) : 0.0f;
            const float rb = SWAP && p.bias && row < p.R ? __ldg(p.bias + row) : 0.0f;
            int okw = 0;
            if (lane == 0) okw = ptx::mbar_wait(&accf_bar[buf], (i >> 1) & 1, err) && *err == 0;
            if (!__shfl_sync(0xffffffffu, okw, 0)) break;
            ptx::tc_fence_after();
            const int nblk = min((BN + 31) / 32, (p.S - s0 + 31) / 32);
            const int last = nblk - 1 - ((nblk - 1 - half) & 1);
            if (last < 0) {  // a warp without a block still releases the accumulator
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(&acce_bar[buf]);
            }
#pragma unroll 1
            for (int c = half; c < nblk; c += 2) {
                const int col0 = s0 + c * 32;
                const int col = min(col0 + lane, p.S - 1);
                __syncwarp();  // the previous block's readers of the tables are done
                tab[lane] = __ldg(p.s_scale + col);
                if (!SWAP) tab[32 + lane] = p.bias ? __ldg(p.bias + col) : 0.0f;
                uint32_t r[32];
                ptx::tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(q * 32) << 16) + buf * C::ACC_COLS + c * 32, r);
                ptx::tmem_ld_wait();
                if (c == last) {
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&acce_bar[buf]);
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 sc = *reinterpret_cast<const float4*>(tab + j);
                    const float4 bi = SWAP ? make_float4(rb, rb, rb, rb) : *reinterpret_cast<const float4*>(tab + 32 + j);
                    const bool hb = p.bias != nullptr;
                    r[j + 0] = __float_as_uint(i8_finish((int)r[j + 0], rs, sc.x, hb, bi.x, p.relu));
                    r[j + 1] = __float_as_uint(i8_finish((int)r[j + 1], rs, sc.y, hb, bi.y, p.relu));
                    r[j + 2] = __float_as_uint(i8_finish((int)r[j + 2], rs, sc.z, hb, bi.z, p.relu));
                    r[j + 3] = __float_as_uint(i8_finish((int)r[j + 3], rs, sc.w, hb, bi.w, p.relu));
                }
                if (SWAP) {  // lanes are adjacent columns of C
                    if (row < p.R) {
                        float* dst = p.C + (int64_t)col0 * p.ldc + row;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (col0 + j < p.S) dst[(int64_t)j * p.ldc] = __uint_as_float(r[j]);
                    }
                } else if (p.tma_store) {
                    if (r0 + q * 32 < p.R) {  // the box parts past R or S are not written
                        if (lane == 0 && stored) ptx::bulk_wait_read<0>();
                        __syncwarp();
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
                        stored = true;
                    }
                } else {  // transpose through shared memory: one 128-byte row segment a store
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 32; ++j)  // word j of row `lane` at j ^ lane: no bank conflicts either way
                        reinterpret_cast<uint32_t*>(blk)[lane * 32 + (j ^ lane)] = r[j];
                    __syncwarp();
                    if (col0 + lane < p.S)
                        for (int j = 0; j < 32; ++j)
                            if (r0 + q * 32 + j < p.R)
                                p.C[(int64_t)(r0 + q * 32 + j) * p.ldc + col0 + lane] =
                                    __uint_as_float(reinterpret_cast<uint32_t*>(blk)[j * 32 + (lane ^ j)]);
                    __syncwarp();
                }
            }
        }
        if (lane == 0 && stored) ptx::bulk_wait_all();  // C is written before the CTA exits
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

template <class Cf, bool SWAP>
static int launch(const CUtensorMap& r, const CUtensorMap& s, const CUtensorMap& c, const Params& p, cudaStream_t st) {
    static bool attr_set[64] = {};
    static std::mutex mu;
    int dev = 0;
    cudaGetDevice(&dev);
    {
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 0 && dev < 64 && !attr_set[dev]) {
            if (cudaFuncSetAttribute(gemm_i8_tc_kernel<Cf, SWAP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     Cf::SMEM_BYTES) != cudaSuccess)
                return set_status(JST_ERR_CUDA, "cudaFuncSetAttribute(gemm_i8_tc_kernel) failed");
            attr_set[dev] = true;
        }
    }
    const unsigned grid = (unsigned)std::min<int64_t>((int64_t)p.tiles_r * p.tiles_s, sm_count());
    ProfScope prof(st, KID_GEMM_I8);
    if (launch_dependent(gemm_i8_tc_kernel<Cf, SWAP>, dim3(grid), dim3(THREADS), Cf::SMEM_BYTES, st, r, s, c, p) !=
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

static int run_aligned(const I8Args& a, cudaStream_t s) {
    Params p{};
    p.K = a.K;
    p.C = a.C; p.ldc = a.ldc;
    p.bias = a.bias; p.relu = a.relu;
    p.err = device_error_word();
    const bool swap = a.M <= 64;
    int bn;
    if (swap) {
        bn = a.M <= 16 ? 16 : a.M <= 32 ? 32 : 64;
    } else {
        // the widest tile that still gives every SM one
        const int64_t rows = (a.M + BM - 1) / BM, sms = sm_count();
        bn = rows * ((a.N + 255) / 256) >= sms ? 256 : rows * ((a.N + 127) / 128) >= sms ? 128 : 64;
    }
    const int8_t *r = swap ? a.B : a.A, *q = swap ? a.A : a.B;
    const int64_t ldr = swap ? a.ldb : a.lda, lds = swap ? a.lda : a.ldb;
    p.R = swap ? a.N : a.M;
    p.S = swap ? a.M : a.N;
    p.r_scale = swap ? a.b_scale : a.a_scale;
    p.s_scale = swap ? a.a_scale : a.b_scale;
    p.tiles_r = (p.R + BM - 1) / BM;
    p.tiles_s = (p.S + bn - 1) / bn;
    if ((int64_t)p.tiles_r * p.tiles_s > 0x7fffffff) return set_status(JST_ERR_ARG, "gemm_i8: too many tiles");
    const int64_t one = ((int64_t)a.K + 15) / 16 * 16;  // the pitch of a single row is never used
    CUtensorMap mr, ms, mc;
    if (!make_map(&mr, r, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, p.R, p.R == 1 ? one : ldr, BM) ||
        !make_map(&ms, q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, p.S, p.S == 1 ? one : lds, bn))
        return set_status(JST_ERR_CUDA, "cuTensorMapEncodeTiled failed");
    mc = mr;  // not read unless tma_store
    p.tma_store = !swap && (reinterpret_cast<uintptr_t>(a.C) & 15) == 0 && (a.ldc & 3) == 0 &&
                  make_map(&mc, a.C, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, a.N, a.M, a.ldc, 32);
    if (swap) {
        if (bn == 16) return launch<Cfg<16, 8>, true>(mr, ms, mc, p, s);
        if (bn == 32) return launch<Cfg<32, 8>, true>(mr, ms, mc, p, s);
        return launch<Cfg<64, 6>, true>(mr, ms, mc, p, s);
    }
    if (bn == 256) return launch<Cfg<256, 4>, false>(mr, ms, mc, p, s);
    if (bn == 128) return launch<Cfg<128, 5>, false>(mr, ms, mc, p, s);
    return launch<Cfg<64, 6>, false>(mr, ms, mc, p, s);
}

}  // namespace i8

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
