// sq_mm.cu -- 8-bit matrix product with a scale per token and per channel:
//     out[i, j] = float(sum_t a[i, t] * b[j, t]) * a_scale[i] * b_scale[j] + bias[j]
// a [m, k] and b [n, k] int8, both with k innermost.  The sum is exact in 32
// bits (k < 2^17); the scaling and the bias are fp32 and each output is
// rounded once more, to its type.
#include <algorithm>

#include "launch.h"
#include "sq.cuh"
#include "tc.cuh"

namespace isb {

namespace {

template <typename T>
__device__ __forceinline__ void mm_emit(T* out, int acc, float sa, float sb, float bias) {
    sq_round(__fmaf_rn((float)acc * sa, sb, bias), *out);
}

// ---- tiles on the CUDA cores: any alignment --------------------------------
// 64 x 64 outputs per block of 256 threads, 4 x 4 each by __dp4a; 64 bytes of k
// per step through shared memory, stored by words of 4 k with the rows beside
// each other (row index fastest), so that the threads of a warp read
// neighbouring words.
constexpr int kTile = 64, kStep = 64;

__device__ __forceinline__ uint32_t mm_word(const int8_t* row, int t, int k, bool fast) {
    if (fast && t + 4 <= k) return *reinterpret_cast<const uint32_t*>(row + t);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (t + i < k) w |= (uint32_t)(uint8_t)row[t + i] << (8 * i);
    return w;
}

template <typename T>
__global__ void __launch_bounds__(256) mm_tile_kernel(SqMatmul p, int fast_a, int fast_b, int tiles_n) {
    __shared__ uint32_t sa[kStep / 4][kTile + 1], sb[kStep / 4][kTile + 1];
    const int64_t i0 = (int64_t)(blockIdx.x / tiles_n) * kTile, j0 = (int64_t)(blockIdx.x % tiles_n) * kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int t0 = 0; t0 < p.k; t0 += kStep) {
#pragma unroll
        for (int u = 0; u < kTile * kStep / 4 / 256; ++u) {
            const int w = threadIdx.x + 256 * u, r = w / (kStep / 4), c = w % (kStep / 4);
            sa[c][r] = i0 + r < p.m ? mm_word(p.a + (i0 + r) * p.lda, t0 + 4 * c, p.k, fast_a) : 0u;
            sb[c][r] = j0 + r < p.n ? mm_word(p.b + (j0 + r) * p.ldb, t0 + 4 * c, p.k, fast_b) : 0u;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kStep / 4; ++c) {
            int av[4], bv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) av[i] = (int)sa[c][ty + 16 * i];
#pragma unroll
            for (int j = 0; j < 4; ++j) bv[j] = (int)sb[c][tx + 16 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
        }
        __syncthreads();
    }
    T* out = static_cast<T*>(p.out);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t col = j0 + tx + 16 * j;
        if (col >= p.n) continue;
        const float s = p.b_scale[col], bias = p.bias ? p.bias[col] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = i0 + ty + 16 * i;
            if (row < p.m) mm_emit(out + row * p.ldo + col, acc[i][j], p.a_scale[row], s, bias);
        }
    }
}

// ---- tiles on the tensor cores: 16-byte aligned rows ------------------------
// tcgen05.mma kind::i8, s8 x s8 summed exactly in s32 in tensor memory.  The
// channels (rows of b) are the MMA's M, 128 a tile, and the tokens (rows of a)
// its N, NT a tile, so that 1 to 256 tokens fit one tile without padding to
// 128, and accumulator lane i is channel i: the 32 lanes of an epilogue warp
// store 32 neighbouring outputs of one token with no exchange between them.
//
// A CTA takes tiles t = blockIdx.x, + gridDim.x, ...:
//   warp 0      one lane issues the tensor copies, 128 bytes of k of the tile's
//               rows of b and a per stage, 128-byte swizzled, through tensor
//               maps over this GPU's memory (no multicast); rows and bytes past
//               the ends read as zeros;
//   warp 1      allocates tensor memory; one lane issues the MMAs (32 bytes of
//               k each) into one of two accumulators of NT columns;
//   warps 2..   epilogue: scales, bias, rounding and stores, while the next
//               tile's MMAs run.
// Every wait is bounded; after a wait that gives up the CTA's remaining outputs are NaN.
constexpr int kMmM = 128, kMmK = 128;

template <int NT>
struct MmCfg {
    static constexpr int kStage = (kMmM + NT) * kMmK;
    static constexpr int kFit = (227 * 1024 - 1024 - 4096) / kStage;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr int kEpi = NT >= 64 ? 8 : 4;                 // epilogue warps
    static constexpr int kThreads = 64 + 32 * kEpi;
    static constexpr int kCols = 2 * NT;                          // tensor-memory columns
    static constexpr int kHalf = NT / (kEpi / 4);                 // columns of an epilogue warp
    static constexpr int kChunk = kHalf < 32 ? kHalf : 32;
    static constexpr size_t kSmem = (size_t)kStage * kStages + 1024;
};

// tile t of tn channel tiles x tm token tiles: bands of 8 token tiles, so that
// the CTAs at work share rows of both operands in L2
__device__ __forceinline__ void mm_place(int64_t t, int tn, int tm, int& ct, int& tt) {
    const int64_t per = (int64_t)8 * tn;
    const int band = (int)(t / per);
    const int w = min(8, tm - 8 * band);
    const uint32_t r = (uint32_t)(t - band * per);               // below 8 * 2^24
    ct = (int)(r / (uint32_t)w);
    tt = 8 * band + (int)(r - (uint32_t)ct * (uint32_t)w);
}

template <typename T, int NT>
__global__ void __launch_bounds__(MmCfg<NT>::kThreads, 1)
    mm_tc_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a, SqMatmul p,
                 int tn, int tm) {
    using C = MmCfg<NT>;
    extern __shared__ unsigned char sm_raw[];
    unsigned char* sm =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~uintptr_t(1023));
    __shared__ __align__(8) uint64_t bar_full[C::kStages];
    __shared__ __align__(8) uint64_t bar_empty[C::kStages];
    __shared__ __align__(8) uint64_t bar_af[2];
    __shared__ __align__(8) uint64_t bar_ae[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    __shared__ __align__(16) float s_scale[C::kEpi][C::kChunk];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const volatile int* vfail = &s_fail;
    const int64_t tiles = (int64_t)tn * tm;
    const int kblocks = (p.k + kMmK - 1) / kMmK;

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(C::kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bar_af[a], 1);
            mbar_init(&bar_ae[a], C::kEpi);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        s_fail = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp == 0) {
        if (lane == 0) {
            int64_t g = 0;                                       // stages filled so far
            for (int64_t t = blockIdx.x; t < tiles && !*vfail; t += gridDim.x) {
                int ct, tt;
                mm_place(t, tn, tm, ct, tt);
                for (int kb = 0; kb < kblocks; ++kb, ++g) {
                    const int s = (int)(g % C::kStages);
                    if (g >= C::kStages &&
                        !mbar_wait_timed(&bar_empty[s], (uint32_t)((g / C::kStages - 1) & 1), vfail)) {
                        s_fail = 1;
                        break;
                    }
                    unsigned char* st = sm + (size_t)s * C::kStage;
                    mbar_arrive_expect(&bar_full[s], C::kStage);
                    tma_load_2d(st, &map_b, kb * kMmK, ct * kMmM, &bar_full[s]);
                    tma_load_2d(st + kMmM * kMmK, &map_a, kb * kMmK, tt * NT, &bar_full[s]);
                }
            }
            // the copies in flight land before the CTA's shared memory is released
            for (int64_t i = g > C::kStages ? g - C::kStages : 0; i < g; ++i)
                mbar_wait_timed(&bar_full[i % C::kStages], (uint32_t)((i / C::kStages) & 1), nullptr);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_idesc_s8(kMmM, NT);
            int64_t g = 0, n = 0;                                // stages read, tiles done
            for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
                const int a = (int)(n & 1);
                bool ok = n < 2 || mbar_wait_timed(&bar_ae[a], (uint32_t)((n / 2 - 1) & 1), vfail);
                const uint32_t dacc = tmem + (uint32_t)(a * NT);
                for (int kb = 0; ok && kb < kblocks; ++kb, ++g) {
                    const int s = (int)(g % C::kStages);
                    ok = mbar_wait_timed(&bar_full[s], (uint32_t)((g / C::kStages) & 1), vfail);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t b_addr = smem_u32(sm + (size_t)s * C::kStage);
                    const uint32_t a_addr = b_addr + kMmM * kMmK;
                    const int steps = min(4, (p.k - kb * kMmK + 31) / 32);
                    for (int kk = 0; kk < steps; ++kk) {
                        const uint64_t bd = umma_smem_desc_sw128(b_addr + 32 * kk);
                        const uint64_t ad = umma_smem_desc_sw128(a_addr + 32 * kk);
                        const uint32_t acc = kb | kk ? 1u : 0u;
                        asm volatile(
                            "{\n .reg .pred pa;\n setp.ne.b32 pa, %4, 0;\n"
                            " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, pa;\n}" ::"r"(dacc),
                            "l"(bd), "l"(ad), "r"(idesc), "r"(acc)
                            : "memory");
                    }
                    tc_commit(&bar_empty[s]);
                }
                if (!ok) {
                    s_fail = 1;
                    break;
                }
                tc_commit(&bar_af[a]);
            }
            // the MMAs in flight are done before tensor memory and the stages are released
            const int64_t last = n - 1;
            if (n > 0) mbar_wait_timed(&bar_af[last & 1], (uint32_t)((last / 2) & 1), nullptr);
            for (int64_t i = g > C::kStages ? g - C::kStages : 0; i < g; ++i)
                mbar_wait_timed(&bar_empty[i % C::kStages], (uint32_t)((i / C::kStages) & 1), nullptr);
        }
        __syncwarp();
    } else {
        const int ew = warp - 2, quarter = warp & 3, part = ew >> 2;
        float* sc = s_scale[ew];
        T* out = static_cast<T*>(p.out);
        int64_t n = 0;
        bool ok = true;
        for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, ++n) {
            int ct, tt;
            mm_place(t, tn, tm, ct, tt);
            const int a = (int)(n & 1);
            const int64_t ch = (int64_t)ct * kMmM + quarter * 32 + lane;
            const bool in = ch < p.n;
            const float sb = in ? p.b_scale[ch] : 0.f;
            const float bias = in && p.bias ? p.bias[ch] : 0.f;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_timed(&bar_af[a], (uint32_t)((n / 2) & 1), vfail));
            if (!ok && lane == 0) s_fail = 1;
            tc_fence_after();
            for (int c = 0; c < C::kHalf; c += C::kChunk) {
                const int64_t tok = (int64_t)tt * NT + part * C::kHalf + c;
                uint32_t v[C::kChunk];
                if (ok) {
                    const uint32_t ta = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(a * NT + part * C::kHalf + c);
                    if constexpr (C::kChunk == 32) tmem_ld32(ta, v);
                    else tmem_ld16(ta, v);
                }
                if (c + C::kChunk == C::kHalf) {                 // the accumulator is in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_ae[a]);
                }
                const int cnt = (int)min((int64_t)C::kChunk, p.m - tok);
                if (cnt <= 0) continue;
                if (lane < C::kChunk) sc[lane] = lane < cnt ? (ok ? p.a_scale[tok + lane] : __int_as_float(0x7fffffff)) : 0.f;
                __syncwarp();
                T* o = out + tok * p.ldo + ch;
                if (in) {
#pragma unroll
                    for (int j = 0; j < C::kChunk; ++j) {
                        if (j < cnt) mm_emit(o, (int)v[j], sc[j], sb, bias);
                        o += p.ldo;
                    }
                }
                __syncwarp();
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols) : "memory");
}

// the tensor map of int8 rows [n, k], ld bytes apart, read by boxes of 128 bytes x `box` rows
cudaError_t mm_map(const int8_t* rows, int64_t n, int k, int64_t ld, int box, CUtensorMap* map) {
    using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                       const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                       CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    const auto fn = reinterpret_cast<EncodeTiledFn>(encode_tiled_entry());
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)n};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t boxes[2] = {(cuuint32_t)kMmK, (cuuint32_t)box};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(rows), dims, strides, boxes, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

template <typename T, int NT>
cudaError_t launch_tc(const SqMatmul& p, cudaStream_t st) {
    using C = MmCfg<NT>;
    CUtensorMap map_b, map_a;
    cudaError_t e = mm_map(p.b, p.n, p.k, p.ldb, kMmM, &map_b);
    if (!e) e = mm_map(p.a, p.m, p.k, p.lda, NT, &map_a);
    if (!e) e = cudaFuncSetAttribute(mm_tc_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e) return e;
    const int tn = (int)((p.n + kMmM - 1) / kMmM), tm = (int)((p.m + NT - 1) / NT);
    const int grid = (int)std::min<int64_t>((int64_t)tn * tm, sm_count());
    note_launch();
    mm_tc_kernel<T, NT><<<grid, C::kThreads, C::kSmem, st>>>(map_b, map_a, p, tn, tm);
    return cudaGetLastError();
}

bool rows_aligned(const void* p, int64_t ld, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0 && ld % a == 0; }

template <typename T>
cudaError_t launch_mm(const SqMatmul& p, cudaStream_t st) {
    if (rows_aligned(p.a, p.lda, 16) && rows_aligned(p.b, p.ldb, 16)) {
        if (p.m <= 16) return launch_tc<T, 16>(p, st);
        if (p.m <= 32) return launch_tc<T, 32>(p, st);
        if (p.m <= 64) return launch_tc<T, 64>(p, st);
        if (p.m <= 128) return launch_tc<T, 128>(p, st);
        return launch_tc<T, 256>(p, st);
    }
    const int64_t tiles_n = (p.n + kTile - 1) / kTile, tiles_m = (p.m + kTile - 1) / kTile;
    // a grid holds 2^31 - 1 blocks: more tiles go in several launches of whole tile rows
    const int64_t per = std::max<int64_t>(1, ((int64_t(1) << 31) - 1) / tiles_n);
    for (int64_t r = 0; r < tiles_m; r += per) {
        SqMatmul q = p;
        q.a = p.a + r * kTile * p.lda;
        q.a_scale = p.a_scale + r * kTile;
        q.out = static_cast<T*>(p.out) + r * kTile * p.ldo;
        q.m = std::min<int64_t>(p.m - r * kTile, per * kTile);
        const int64_t rows = (q.m + kTile - 1) / kTile;
        note_launch();
        mm_tile_kernel<T><<<(unsigned)(rows * tiles_n), 256, 0, st>>>(
            q, rows_aligned(q.a, q.lda, 4), rows_aligned(q.b, q.ldb, 4), (int)tiles_n);
        const cudaError_t e = cudaGetLastError();
        if (e) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t sq_matmul(const SqMatmul& p, int out_type, cudaStream_t st) {
    if (p.m == 0 || p.n == 0) return cudaSuccess;
    if (out_type == kSqF32) return launch_mm<float>(p, st);
    if (out_type == kSqF16) return launch_mm<__half>(p, st);
    return launch_mm<__nv_bfloat16>(p, st);
}

}  // namespace isb
