// sq_mm.cu -- 8-bit matrix product with a scale per token and per channel:
//     out[i, j] = float(sum_t a[i, t] * b[j, t]) * a_scale[i] * b_scale[j] + bias[j]
// a [m, k] and b [n, k] int8, both with k innermost.  The sum is exact in 32
// bits (k < 2^17); the scaling and the bias are fp32 and each output is
// rounded once more, to its type.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "launch.h"
#include "sq.cuh"
#include "tc.cuh"

namespace isb {

namespace {

template <typename T>
__device__ __forceinline__ void mm_emit(T* out, int acc, float sa, float sb, float bias) {
    sq_round(__fmaf_rn((float)acc * sa, sb, bias), *out);
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

bool rows_aligned(const void* p, int64_t ld, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0 && ld % a == 0; }

// ---- up to 4 tokens: dot products on the CUDA cores ------------------------
// With so few tokens every byte of b is used a handful of times, and the
// product is the time to read b.  The tokens' codes lie in shared memory (each
// block quantises them itself when they come as floating rows: one launch in
// all).  A team of TEAM lanes takes R rows of b, 16 bytes a lane and row at a
// time, so that several loads are in flight and each word of the tokens read
// from shared memory serves R rows.  The teams' sums are joined by exchanging
// halves: a lane ends up with its own outputs, V / TEAM of the V = MT * R.
// 1 x 65536 x 128 with fp32 queries: 4.7 us (11.9 us as two launches, tiles for
// the product); 1 x 1M x 128: 28.5 us, 4.8 TB/s.
constexpr int kDotThreads = 256;
constexpr int kDotTokens = 4;
constexpr size_t kDotSmem = 72 * 1024;          // most shared memory for the tokens: three blocks an SM

template <int MT, int R>
constexpr int kDotCtas = MT * R <= 4 ? 3 : 2;   // blocks an SM that the registers of MT * R sums allow

struct MmDot {
    SqMatmul p;
    const void* x;                              // floating tokens (null: p.a, p.a_scale)
    int64_t ldx;
    int x_type, out_type, x_vec;
    int kp;                                     // bytes of a token's codes in shared memory
};

// quantises one floating row of k values into shared memory (one scale), by the whole block
template <typename T, int MODE>
__device__ __forceinline__ void dot_quantise(const T* x, int k, uint8_t* codes, float* scale, uint32_t* s_top) {
    constexpr int E = sq_chunk<T, 8, MODE>();
    uint32_t top = 0;
    SqLoad<T, MODE, E> v;
    const SqSpan span{};                                         // (not used in these modes)
    for (int e0 = threadIdx.x * E; e0 < k; e0 += kDotThreads * E) {
        v.issue(x, e0, k, span);
        v.take(x, e0, k, span).top(top);
    }
    top = __reduce_max_sync(0xffffffffu, __float_as_uint(sq_top<T>(top)));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
    top = 0;
#pragma unroll
    for (int w = 0; w < kDotThreads / 32; ++w) top = max(top, s_top[w]);
    const SqScale s = sq_scale<8>(__uint_as_float(top));
    for (int e0 = threadIdx.x * E; e0 < k; e0 += kDotThreads * E) {
        v.issue(x, e0, k, span);
        sq_store<T, 8, MODE, E>(codes, e0, k, v.take(x, e0, k, span), s);
    }
    if (threadIdx.x == 0) *scale = s.scale;
}
template <typename T>
__device__ __forceinline__ void dot_quantise(const MmDot& q, int i, uint8_t* codes, float* scale, uint32_t* s_top) {
    const T* x = static_cast<const T*>(q.x) + i * q.ldx;
    if (q.x_vec) dot_quantise<T, kSqVec>(x, q.p.k, codes, scale, s_top);
    else dot_quantise<T, kSqSingle>(x, q.p.k, codes, scale, s_top);
}

// sums acc[0 .. N) over the 2 O lanes that differ in the bits below 2 O; the lane's
// share, N / (2 O) values (or one, held by several lanes), is left in
// acc[0 ..): values from the returned index on
template <int N, int O, int V>
__device__ __forceinline__ int dot_join(int (&acc)[V], int tl) {
    if constexpr (O == 0) return 0;
    else if constexpr (N > 1) {
        const bool up = (tl & O) != 0;
#pragma unroll
        for (int q = 0; q < N / 2; ++q) {
            const int give = up ? acc[q] : acc[q + N / 2], keep = up ? acc[q + N / 2] : acc[q];
            acc[q] = keep + __shfl_xor_sync(0xffffffffu, give, O);
        }
        return (up ? N / 2 : 0) + dot_join<N / 2, O / 2, V>(acc, tl);
    } else {
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], O);
        return dot_join<1, O / 2, V>(acc, tl);
    }
}

template <int MT, int TEAM, int R, bool ALIGNED>
__global__ void __launch_bounds__(kDotThreads, kDotCtas<MT, R>) mm_dot_kernel(MmDot q) {
    constexpr int V = MT * R, NV = V / TEAM > 0 ? V / TEAM : 1;
    constexpr int TEAMS = kDotThreads / TEAM;
    extern __shared__ __align__(16) uint8_t s_a[];               // [MT][kp]
    __shared__ float s_scale[MT];
    __shared__ uint32_t s_top[kDotThreads / 32];
    const SqMatmul& p = q.p;
    const int m = (int)p.m;
    const int tl = threadIdx.x % TEAM, team = threadIdx.x / TEAM;

    for (int i = 0; i < MT; ++i) {
        uint8_t* row = s_a + (size_t)i * q.kp;
        if (i >= m) {
            for (int t = threadIdx.x; t < q.kp / 16; t += kDotThreads)
                reinterpret_cast<uint4*>(row)[t] = make_uint4(0u, 0u, 0u, 0u);
            if (threadIdx.x == 0) s_scale[i] = 0.f;
        } else if (q.x) {
            for (int t = p.k + threadIdx.x; t < q.kp; t += kDotThreads) row[t] = 0;
            if (q.x_type == kSqF32) dot_quantise<float>(q, i, row, s_scale + i, s_top);
            else if (q.x_type == kSqF16) dot_quantise<__half>(q, i, row, s_scale + i, s_top);
            else dot_quantise<__nv_bfloat16>(q, i, row, s_scale + i, s_top);
        } else {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(p.a), hi = lo + (m - 1) * p.lda + p.k;
            const uintptr_t a = lo + i * p.lda;
            for (int t = threadIdx.x; t < q.kp / 16; t += kDotThreads) {
                SqBytes<false> w;
                w.issue(a + 16 * t, a + p.k, lo, hi);
                reinterpret_cast<uint4*>(row)[t] = w.take(a + 16 * t, a + p.k, lo, hi);
            }
            if (threadIdx.x == 0) s_scale[i] = p.a_scale[i];
        }
    }
    __syncthreads();

    const uintptr_t lo = reinterpret_cast<uintptr_t>(p.b), hi = lo + (p.n - 1) * p.ldb + p.k;
    const int64_t step = (int64_t)gridDim.x * (TEAMS * R);
    // the loop bound is the same for a warp's teams: all lanes take part in every exchange
    for (int64_t j0 = (int64_t)blockIdx.x * (TEAMS * R); j0 < p.n; j0 += step) {
        const int64_t j = j0 + team * R;
        uintptr_t b[R], end[R];                                  // a row past the last one is empty
#pragma unroll
        for (int r = 0; r < R; ++r) {
            b[r] = lo + (j + r < p.n ? j + r : 0) * p.ldb;
            end[r] = b[r] + (j + r < p.n ? p.k : 0);
        }
        int acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0;
#pragma unroll R <= 2 ? 8 / R : 2
        for (int t = tl * 16; t < q.kp; t += TEAM * 16) {
            SqBytes<ALIGNED> raw[R];
#pragma unroll
            for (int r = 0; r < R; ++r) raw[r].issue(b[r] + t, end[r], lo, hi);
            uint4 w[R];
#pragma unroll
            for (int r = 0; r < R; ++r) w[r] = raw[r].take(b[r] + t, end[r], lo, hi);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const uint4 a = *reinterpret_cast<const uint4*>(s_a + (size_t)i * q.kp + t);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    int s = acc[i * R + r];
                    s = __dp4a((int)a.x, (int)w[r].x, s);
                    s = __dp4a((int)a.y, (int)w[r].y, s);
                    s = __dp4a((int)a.z, (int)w[r].z, s);
                    acc[i * R + r] = __dp4a((int)a.w, (int)w[r].w, s);
                }
            }
        }
        const int v0 = dot_join<V, TEAM / 2, V>(acc, tl);
        if (V < TEAM && (tl & (TEAM / V - 1)) != 0) continue;    // one of the lanes that hold a value stores it
#pragma unroll
        for (int e = 0; e < NV; ++e) {
            const int i = (v0 + e) / R;
            const int64_t col = j + (v0 + e) % R;
            if (i >= m || col >= p.n) continue;
            const float sb = p.b_scale[col], bias = p.bias ? p.bias[col] : 0.f;
            const int64_t at = i * p.ldo + col;
            if (q.out_type == kSqF32) mm_emit(static_cast<float*>(p.out) + at, acc[e], s_scale[i], sb, bias);
            else if (q.out_type == kSqF16) mm_emit(static_cast<__half*>(p.out) + at, acc[e], s_scale[i], sb, bias);
            else mm_emit(static_cast<__nv_bfloat16*>(p.out) + at, acc[e], s_scale[i], sb, bias);
        }
    }
}

template <int MT, int TEAM, int R, bool ALIGNED>
cudaError_t go_dot(const MmDot& q, cudaStream_t st) {
    const size_t smem = (size_t)MT * q.kp;
    if (smem > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(mm_dot_kernel<MT, TEAM, R, ALIGNED>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kDotSmem);
        if (e) return e;
    }
    const int64_t per = kDotThreads / TEAM * R;
    const int grid = (int)std::min<int64_t>((q.p.n + per - 1) / per, (int64_t)sm_count() * kDotCtas<MT, R>);
    note_launch();
    mm_dot_kernel<MT, TEAM, R, ALIGNED><<<grid, kDotThreads, smem, st>>>(q);
    return cudaGetLastError();
}

// As many lanes a row as its 16-byte pieces need: 2, 8 or 16, else the warp.  A
// single token takes fewer rows a warp where there are few rows, so that all
// SMs have warps (1 x 4096 x 4096: 9.3 us with 4 rows, 7.3 us with 2).
template <int MT, bool ALIGNED>
cudaError_t by_team(const MmDot& q, cudaStream_t st) {
    if (q.kp <= 32) return go_dot<MT, 2, 4, ALIGNED>(q, st);
    if (q.kp <= 128) return go_dot<MT, 8, MT == 1 ? 8 : 4, ALIGNED>(q, st);
    if (q.kp <= 256) return go_dot<MT, 16, MT == 1 ? 8 : 4, ALIGNED>(q, st);
    if constexpr (MT == 1) {
        if (q.p.n < 4096) return go_dot<MT, 32, 1, ALIGNED>(q, st);
        if (q.p.n < 10000) return go_dot<MT, 32, 2, ALIGNED>(q, st);
    }
    return go_dot<MT, 32, 4, ALIGNED>(q, st);
}

// bytes of a token's codes that a team's lanes read: whole steps of the team
int dot_kp(int k) {
    const int step = k <= 32 ? 32 : k <= 128 ? 128 : k <= 256 ? 256 : 512;
    return (k + step - 1) / step * step;
}

bool dot_usable(const SqMatmul& p) {
    const int mt = p.m == 1 ? 1 : kDotTokens;
    return p.m <= kDotTokens && (size_t)mt * dot_kp(p.k) <= kDotSmem;
}

cudaError_t launch_dot(MmDot q, cudaStream_t st) {
    q.kp = dot_kp(q.p.k);
    const bool al = rows_aligned(q.p.b, q.p.ldb, 16);
    if (q.p.m == 1) return al ? by_team<1, true>(q, st) : by_team<1, false>(q, st);
    return al ? by_team<kDotTokens, true>(q, st) : by_team<kDotTokens, false>(q, st);
}

// ---- tiles on the tensor cores ---------------------------------------------
// tcgen05.mma kind::i8, s8 x s8 summed exactly in s32 in tensor memory.  The
// channels (rows of b) are the MMA's M, 128 a tile, and the tokens (rows of a)
// its N, NT a tile, so that 1 to 256 tokens fit one tile without padding to
// 128, and accumulator lane i is channel i: the 32 lanes of an epilogue warp
// store 32 neighbouring outputs of one token with no exchange between them.
//
// A unit of work is a tile, or, with `split` > 1, one of the `split` parts of a
// tile's k; a CTA takes the units blockIdx.x, + gridDim.x, ... (one unit each when
// k is split):
//   warp 0      one lane issues the tensor copies, 128 bytes of k of the tile's
//               rows of b and a per stage, 128-byte swizzled, through tensor
//               maps over this GPU's memory (no multicast); rows and bytes past
//               the ends read as zeros;
//   warp 1      allocates tensor memory; one lane issues the MMAs (32 bytes of
//               k each) into one of two accumulators of NT columns;
//   warps 2..   epilogue: scales, bias, rounding and stores, while the next
//               tile's MMAs run.
// The parts of a split tile are the CTAs of one cluster: each leaves its sums in
// its shared memory and adds up, over the cluster, the columns that fall to
// it (whole numbers: the order does not matter).
// Every wait on a barrier in memory is bounded; a CTA in which one gives up raises
// g_mm_gave_up (its outputs are not valid then: what it still stores is NaN
// mostly), lets its copies and MMAs in flight end, and returns.
constexpr int kMmM = 128, kMmK = 128;

template <int NT>
struct MmCfg {
    static constexpr int kStage = (kMmM + NT) * kMmK;
    static constexpr int kEpi = NT >= 256 ? 16 : NT >= 64 ? 8 : 4;   // epilogue warps
    static constexpr int kThreads = 64 + 32 * kEpi;
    static constexpr int kCtas = NT <= 128 ? 2 : 1;               // resident per SM
    static constexpr int kCols = 2 * NT;                          // tensor-memory columns
    static constexpr int kHalf = NT / (kEpi / 4);                 // columns of an epilogue warp
    static constexpr int kChunk = kHalf < 32 ? kHalf : 32;
    static constexpr int kStatic = kEpi * kHalf * 4 + 1024;       // static arrays
    static constexpr int kStages = (227 * 1024 / kCtas - 1024 - 1024 - kStatic) / kStage;   // 1 KB to align, 1 KB of the system's
    static constexpr size_t kSmem = (size_t)kStage * kStages + 1024;
    static_assert(kStages >= 2 && (size_t)kMmM * NT * 4 <= (size_t)kStage * kStages, "a split tile's sums fit the stages");
};

// tile t of tn channel tiles x tm token tiles: bands of 8 token tiles, so that
// the CTAs at work share rows of both operands in L2.  32-bit divisions: 64-bit
// ones took a third of the epilogue's instructions at k = 128.
__device__ __forceinline__ void mm_place(uint32_t t, uint32_t tn, uint32_t tm, int& ct, int& tt) {
    const uint32_t per = 8 * tn, band = t / per, w = min(8u, tm - 8 * band), r = t - band * per;
    ct = (int)(r / w);
    tt = (int)(8 * band + r - (uint32_t)ct * w);
}

// set by a product with a wait that gave up, read and cleared by sq_status
__device__ int g_mm_gave_up;

// Wait on an mbarrier phase, suspended, bounded by `limit` ns of wall time; false
// where it gave up, early once *fail is set (fail may be null).  A limit of 0 polls only.
__device__ __forceinline__ bool mm_wait(uint64_t* bar, uint32_t parity, const volatile int* fail, uint32_t limit) {
    if (mbar_try_wait_sleep(bar, parity, min(limit, 20000u))) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        if (fail && *fail) return false;
        const bool over = globaltimer_ns() - t0 >= limit;
        if (mbar_try_wait_sleep(bar, parity, over ? 0u : 20000u)) return true;
        if (over) return false;
    }
}

// The copying and the MMA thread run once per 128 bytes of k, some 500 clocks of
// the tensor core: their place in the ring of stages is counted, not divided
// out (a 64-bit remainder a step made 8192^3 a tenth slower).
struct MmRing {
    uint32_t s = 0, lap = 0;                    // stage, times round the ring
    __device__ __forceinline__ void next(uint32_t stages) {
        if (++s == stages) {
            s = 0;
            ++lap;
        }
    }
};

// waits, for kTCWaitNs each, until every phase of a ring's stages that was begun is over
__device__ __forceinline__ void mm_drain(uint64_t* bars, MmRing r, uint32_t stages) {
    for (uint32_t i = 0; i < stages; ++i) {
        // stage i was last used in lap `lap` where i is before the ring's place, else in the lap before
        if (i < r.s) mm_wait(bars + i, r.lap & 1, nullptr, kTCWaitNs);
        else if (r.lap > 0) mm_wait(bars + i, (r.lap - 1) & 1, nullptr, kTCWaitNs);
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}

// the 32-bit word at shared-memory address `at` of CTA `rank` of the cluster
__device__ __forceinline__ int cluster_load(uint32_t at, int rank) {
    uint32_t remote;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    return v;
}

// the 16 bytes there
__device__ __forceinline__ int4 cluster_load4(uint32_t at, int rank) {
    uint32_t remote;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(remote)
                 : "memory");
    return v;
}

// one MMA: accumulator d, channels' descriptor b, tokens' descriptor a
__device__ __forceinline__ void mm_issue(uint32_t d, uint64_t b, uint64_t a, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred pa;\n setp.ne.b32 pa, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, pa;\n}" ::"r"(d),
        "l"(b), "l"(a), "r"(idesc), "r"(acc)
        : "memory");
}

struct MmTc {
    SqMatmul p;
    int out_type;
    uint32_t tn, tm;            // channel and token tiles, fewer than 2^31 in all
    int split;                  // parts of k (the cluster's size)
    int kb_part;                // 128-byte blocks of k per part
    uint32_t copy_bytes;        // of a stage's two tensor copies
    uint32_t wait_ns;           // how long a wait lasts before it gives up
    bool pair;                  // 2 neighbouring 16-bit outputs may be stored at once
};

// Outputs of an epilogue warp: 32 channels (one a lane, `nch` of them there) of
// `cnt` tokens (at most N) from `o` on (the lane's channel), rows ldo values apart.
//
// With output-bound products (k near 128) the instructions of this loop decide.
// Two tokens are scaled at once by packed fp32 pairs; sums of at most 2^22
// (SMALL: k <= 256) become floats by adding 1.5 * 2^23 as bits, which is exact
// and leaves the slow integer conversion out; and 16-bit outputs (pair: rows
// 4-byte aligned) are exchanged with the neighbouring lane, so that each lane
// stores 2 channels of one token.  Turning the block in shared memory for
// 16-byte stores was slower (fp32 scores of 256 x 1M: 283 against 222 us): its
// round trips wait longer than the stores they save.
template <bool SMALL>
__device__ __forceinline__ float2 mm_scaled(uint32_t v0, uint32_t v1, float2 sa, float sb, float bias) {
    constexpr float kMagic = 12582912.f;
    const float2 f = SMALL ? sq_add2(make_float2(__uint_as_float(0x4b400000u + v0), __uint_as_float(0x4b400000u + v1)),
                                     make_float2(-kMagic, -kMagic))
                           : make_float2((float)(int)v0, (float)(int)v1);
    return sq_fma2(sq_mul2(f, sa), make_float2(sb, sb), make_float2(bias, bias));
}

__device__ __forceinline__ uint32_t mm_pack(float2 r, __half) {
    const __half2 h = __floats2half2_rn(r.x, r.y);
    uint32_t w;
    memcpy(&w, &h, 4);
    return w;
}
__device__ __forceinline__ uint32_t mm_pack(float2 r, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(r.x, r.y);
    uint32_t w;
    memcpy(&w, &h, 4);
    return w;
}

template <typename T, int N, bool SMALL>
__device__ __forceinline__ void mm_block(T* o, int64_t ldo, const uint32_t (&v)[N], const float* sc, int cnt, float sb,
                                         float bias, int nch, int lane, bool pair) {
    if constexpr (sizeof(T) == 2) {
        if (pair && cnt == N && nch >= 32) {
            const int odd = lane & 1;
            o += odd ? ldo - 1 : 0;                              // an odd lane stores the second token
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const uint32_t w = mm_pack(mm_scaled<SMALL>(v[j], v[j + 1], *reinterpret_cast<const float2*>(sc + j), sb,
                                                            bias),
                                           T{});
                const uint32_t x = __shfl_xor_sync(0xffffffffu, w, 1);
                const uint32_t y = __byte_perm(w, x, odd ? 0x3276 : 0x5410);
                *reinterpret_cast<uint32_t*>(o) = y;
                o += 2 * ldo;
            }
            return;
        }
    }
    if (lane >= nch) return;
    if (cnt == N) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float2 r = mm_scaled<SMALL>(v[j], v[j + 1], *reinterpret_cast<const float2*>(sc + j), sb, bias);
            sq_round(r.x, o[0]);
            sq_round(r.y, o[ldo]);
            o += 2 * ldo;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (j < cnt) mm_emit(o, (int)v[j], sc[j], sb, bias);
            o += ldo;
        }
    }
}

template <int N>
__device__ __forceinline__ void mm_block(const MmTc& q, int64_t at, const uint32_t (&v)[N], const float* sc, int cnt,
                                         float sb, float bias, int nch, int lane) {
    auto go = [&](auto* out) {
        using T = std::remove_pointer_t<decltype(out)>;
        if (q.p.k <= 256) mm_block<T, N, true>(out + at, q.p.ldo, v, sc, cnt, sb, bias, nch, lane, q.pair);
        else mm_block<T, N, false>(out + at, q.p.ldo, v, sc, cnt, sb, bias, nch, lane, q.pair);
    };
    if (q.out_type == kSqF32) go(static_cast<float*>(q.p.out));
    else if (q.out_type == kSqF16) go(static_cast<__half*>(q.p.out));
    else go(static_cast<__nv_bfloat16*>(q.p.out));
}

template <int NT>
__global__ void __launch_bounds__(MmCfg<NT>::kThreads, MmCfg<NT>::kCtas)
    mm_tc_kernel(const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_a,
                 const __grid_constant__ MmTc q) {
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
    __shared__ __align__(16) float s_scale[C::kEpi][C::kHalf];
    const SqMatmul& p = q.p;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const volatile int* vfail = &s_fail;
    const int split = q.split, part = split > 1 ? (int)(blockIdx.x % split) : 0;
    const uint32_t t0 = split > 1 ? blockIdx.x / split : blockIdx.x;
    const uint32_t tiles = split > 1 ? t0 + 1 : q.tn * q.tm;              // one past this CTA's last
    const int kb0 = part * q.kb_part;
    const int kb1 = min(kb0 + q.kb_part, (p.k + kMmK - 1) / kMmK);

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
    // what was queued before (the kernel that quantised the tokens) is done from here on
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            MmRing r;
            for (uint32_t t = t0; t < tiles && !*vfail; t += gridDim.x) {
                int ct, tt;
                mm_place(t, q.tn, q.tm, ct, tt);
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (r.lap > 0 && !mm_wait(&bar_empty[r.s], (r.lap - 1) & 1, vfail, q.wait_ns)) {
                        s_fail = 1;
                        break;
                    }
                    unsigned char* st = sm + (size_t)r.s * C::kStage;
                    mbar_arrive_expect(&bar_full[r.s], q.copy_bytes);
                    tma_load_2d(st, &map_b, kb * kMmK, ct * kMmM, &bar_full[r.s]);
                    tma_load_2d(st + kMmM * kMmK, &map_a, kb * kMmK, tt * NT, &bar_full[r.s]);
                    r.next(C::kStages);
                }
            }
            // the copies in flight land before the CTA's shared memory is released
            mm_drain(bar_full, r, C::kStages);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_idesc_s8(kMmM, NT);
            const uint64_t desc0 = umma_smem_desc_sw128(smem_u32(sm));
            const int last = (p.k - (kb1 - 1) * kMmK + 31) / 32;          // MMAs of the last step of k, at least
            MmRing r;
            uint32_t n = 0;                                      // tiles done
            for (uint32_t t = t0; t < tiles; t += gridDim.x, ++n) {
                const uint32_t a = n & 1;
                bool ok = n < 2 || mm_wait(&bar_ae[a], (n / 2 - 1) & 1, vfail, q.wait_ns);
                const uint32_t dacc = tmem + a * NT;
                for (int kb = kb0; ok && kb < kb1; ++kb) {
                    ok = mm_wait(&bar_full[r.s], r.lap & 1, vfail, q.wait_ns);
                    if (!ok) break;
                    tc_fence_after();
                    // descriptor addresses count 16 bytes; one MMA reads 32 bytes of k
                    const uint64_t bd = desc0 + r.s * (C::kStage >> 4), ad = bd + (kMmM * kMmK >> 4);
                    mm_issue(dacc, bd, ad, idesc, kb > kb0);
                    const int steps = kb + 1 == kb1 ? last : 4;
                    if (steps > 1) mm_issue(dacc, bd + 2, ad + 2, idesc, 1);
                    if (steps > 2) mm_issue(dacc, bd + 4, ad + 4, idesc, 1);
                    if (steps > 3) mm_issue(dacc, bd + 6, ad + 6, idesc, 1);
                    tc_commit(&bar_empty[r.s]);
                    r.next(C::kStages);
                }
                if (!ok) {
                    s_fail = 1;
                    break;
                }
                tc_commit(&bar_af[a]);
            }
            // the MMAs in flight are done before tensor memory and the stages are released, and the
            // last commit has arrived where the epilogue does not wait for it any more
            mm_drain(bar_empty, r, C::kStages);
            if (n > 0) mm_wait(&bar_af[(n - 1) & 1], ((n - 1) / 2) & 1, nullptr, kTCWaitNs);
        }
        __syncwarp();
    } else {
        const int ew = warp - 2, quarter = warp & 3, side = ew >> 2;
        float* sc = s_scale[ew];
        uint32_t n = 0;                                          // tiles done
        bool ok = true;
        // a tile's place, scales and bias are found a tile ahead: a load that a
        // chunk of columns waits for is a good part of its time
        constexpr int kSa = (C::kHalf + 31) / 32;
        int ct_next = 0, tt_next = 0;
        float sb_next = 0.f, bias_next = 0.f, sa_next[kSa] = {};
        auto fetch = [&](uint32_t t) {
            mm_place(t, q.tn, q.tm, ct_next, tt_next);
            const int64_t ch = (int64_t)ct_next * kMmM + quarter * 32 + lane;
            if (ch < p.n) {
                sb_next = p.b_scale[ch];
                bias_next = p.bias ? p.bias[ch] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kSa; ++i) {
                const int64_t tok = (int64_t)tt_next * NT + side * C::kHalf + i * 32 + lane;
                sa_next[i] = tok < p.m ? p.a_scale[tok] : 0.f;
            }
        };
        if (t0 < tiles) fetch(t0);
        for (uint32_t t = t0; t < tiles; t += gridDim.x, ++n) {
            const int a = (int)(n & 1), tt = tt_next;
            const int64_t ch = (int64_t)ct_next * kMmM + quarter * 32 + lane;
            const float sb = sb_next, bias = bias_next;
            if (split == 1) {
#pragma unroll
                for (int i = 0; i < kSa; ++i)
                    if (i * 32 + lane < C::kHalf) sc[i * 32 + lane] = sa_next[i];
            }
            if (t + gridDim.x < tiles) fetch(t + gridDim.x);
            if (ok) ok = __all_sync(0xffffffffu, mm_wait(&bar_af[a], (n / 2) & 1, vfail, q.wait_ns));
            if (!ok) {
                if (lane == 0) s_fail = 1;
                for (int i = lane; i < C::kHalf; i += 32) sc[i] = __int_as_float(0x7fffffff);
            }
            __syncwarp();
            tc_fence_after();
            if (split > 1) {
                // this part's sums to shared memory, [column][channel] (the stages
                // are read: the accumulator is done)
                int* x = reinterpret_cast<int*>(sm) + (size_t)side * C::kHalf * kMmM + quarter * 32 + lane;
                for (int c = 0; c < C::kHalf; c += C::kChunk) {
                    uint32_t v[C::kChunk];
                    const uint32_t ta = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(side * C::kHalf + c);
                    if constexpr (C::kChunk == 32) tmem_ld32(ta, v);
                    else tmem_ld16(ta, v);
#pragma unroll
                    for (int j = 0; j < C::kChunk; ++j) x[(size_t)(c + j) * kMmM] = (int)v[j];
                }
                break;
            }
            for (int c = 0; c < C::kHalf; c += C::kChunk) {
                const int64_t tok = (int64_t)tt * NT + side * C::kHalf + c;
                uint32_t v[C::kChunk];
                if (ok) {
                    const uint32_t ta = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(a * NT + side * C::kHalf + c);
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
                mm_block(q, tok * p.ldo + ch, v, sc + c, cnt, sb, bias, (int)min((int64_t)32, p.n - (ch - lane)), lane);
            }
            __syncwarp();                                        // sc is read
        }
    }

    __syncthreads();
    if (tid == 0 && s_fail) g_mm_gave_up = 1;
    if (split > 1) {
        // every part's sums are in its shared memory; column c of the tile falls to part c % split
        cluster_sync();
        int ct, tt;
        mm_place(t0, q.tn, q.tm, ct, tt);
        const int bad = s_fail;
        const uint32_t x = smem_u32(sm), fail_at = smem_u32(&s_fail);
        int any = bad;
        for (int r = 0; r < split; ++r) any |= cluster_load(fail_at, r);
        const int64_t left = p.m - (int64_t)tt * NT;
        const int cols = (int)(left < NT ? left : NT);
        for (int e = tid; e < kMmM / 4 * ((cols - part + split - 1) / split); e += C::kThreads) {
            const int c = part + e / (kMmM / 4) * split, l = e % (kMmM / 4) * 4;      // 4 channels of column c
            int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll 4
            for (int r = 0; r < split; ++r) {
                const int4 v = cluster_load4(x + 4u * (uint32_t)(c * kMmM + l), r);
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            const int64_t ch = (int64_t)ct * kMmM + l, tok = (int64_t)tt * NT + c;
            const float sa = any ? __int_as_float(0x7fffffff) : p.a_scale[tok];
            const int part_sum[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (ch + i >= p.n) break;
                const float sb = p.b_scale[ch + i], bias = p.bias ? p.bias[ch + i] : 0.f;
                const int64_t at = tok * p.ldo + ch + i;
                if (q.out_type == kSqF32) mm_emit(static_cast<float*>(p.out) + at, part_sum[i], sa, sb, bias);
                else if (q.out_type == kSqF16) mm_emit(static_cast<__half*>(p.out) + at, part_sum[i], sa, sb, bias);
                else mm_emit(static_cast<__nv_bfloat16*>(p.out) + at, part_sum[i], sa, sb, bias);
            }
        }
        __syncthreads();
        cluster_sync();                                          // no CTA leaves while its sums are read
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols) : "memory");
}

// the tensor map of int8 rows [n, k], ld bytes apart, in swizzled boxes of 128 bytes x `box` rows
cudaError_t mm_map_rows(const int8_t* rows, int64_t n, int k, int64_t ld, int box, CUtensorMap* map) {
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

// whether 2 neighbouring 16-bit outputs of a row may be stored at once
bool pair_out(const SqMatmul& p, int out_type) { return out_type != kSqF32 && rows_aligned(p.out, 2 * p.ldo, 4); }

// INSITU_SQ_WAIT_NS, read on every call: the limit of a product's waits, at most kTCWaitNs (the default)
uint32_t mm_wait_ns() {
    const char* v = std::getenv("INSITU_SQ_WAIT_NS");
    if (!v || v[0] < '0' || v[0] > '9') return kTCWaitNs;
    return (uint32_t)std::min<unsigned long long>(std::strtoull(v, nullptr, 10), kTCWaitNs);
}

template <int NT>
cudaError_t go_tc(const SqMatmul& p, int out_type, int split, cudaStream_t st) {
    using C = MmCfg<NT>;
    CUtensorMap map_b{}, map_a{};
    // A box has no more rows than its operand: rows that are not there take
    // time to fill in.  What the shared memory holds in their place only reaches
    // accumulators of channels and tokens that are not there either.
    const int box_b = (int)std::min<int64_t>(kMmM, p.n), box_a = (int)std::min<int64_t>(NT, p.m);
    cudaError_t e = mm_map_rows(p.b, p.n, p.k, p.ldb, box_b, &map_b);
    if (!e) e = mm_map_rows(p.a, p.m, p.k, p.lda, box_a, &map_a);
    if (!e) e = cudaFuncSetAttribute(mm_tc_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e) return e;
    MmTc q{};
    q.p = p;
    q.out_type = out_type;
    q.pair = pair_out(p, out_type);
    q.copy_bytes = (uint32_t)(box_a + box_b) * kMmK;
    q.wait_ns = mm_wait_ns();
    q.tn = (uint32_t)((p.n + kMmM - 1) / kMmM);
    q.tm = (uint32_t)((p.m + NT - 1) / NT);
    if ((int64_t)q.tn * q.tm >= int64_t(1) << 31) return cudaErrorInvalidValue;
    const int kb = (p.k + kMmK - 1) / kMmK;
    q.kb_part = (kb + split - 1) / split;
    q.split = (kb + q.kb_part - 1) / q.kb_part;                  // every part has work
    const int64_t tiles = (int64_t)q.tn * q.tm;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(q.split > 1 ? tiles * q.split : std::min<int64_t>(tiles, (int64_t)sm_count() * C::kCtas)));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)q.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    // the kernel may start, and set itself up, while the one before it ends
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    note_launch();
    return cudaLaunchKernelEx(&cfg, mm_tc_kernel<NT>, map_b, map_a, q);
}

// Which tile and how many parts of k: the least of an estimate, in us, that was
// fitted to sweeps of 30 shapes from 16 x 512 x 8192 to 256 x 1M x 128 on a B200
// (most choices are within a tenth of the best of their sweep).  An SM draws
// what it has in flight per 1.6 us of latency under load, the stages of its
// resident CTAs, at most 130 bytes a ns; b comes from HBM at 5 TB/s or from L2;
// a unit's epilogue costs 0.35 us and 1 us per 13000 outputs; a split costs a
// cluster launch, two cluster barriers and the sums' way through shared
// memory, and CTAs beyond those that are resident start anew.  With few tiles a
// split is worth much: 64 x 256 x 16384 takes 11.3 us in 8 parts, 46 us whole;
// 256 x 4096 x 4096 14.9 and 17.3 us.
struct MmPick {
    int nt, split;
    double us;
};

template <int NT>
void mm_estimate(const SqMatmul& p, int sms, MmPick& best) {
    using C = MmCfg<NT>;
    if (NT > 16 && NT / 2 >= p.m) return;                        // a smaller tile holds all tokens
    const double tm = (double)((p.m + NT - 1) / NT), tiles = (double)((p.n + kMmM - 1) / kMmM) * tm;
    const int kb = (p.k + kMmK - 1) / kMmK;
    const double rows = std::min<int64_t>(kMmM, p.n) + std::min<int64_t>(NT, p.m), epi = 0.35 + NT * kMmM / 13000.0;
    for (int split = 1; split <= 8; split *= 2) {
        if (split > 1 && (kb < 2 * split || tiles * split > 8.0 * sms)) break;
        const double per_sm = std::ceil(tiles * split / sms), ctas = std::min<double>(C::kCtas, per_sm);
        const int kb_part = (kb + split - 1) / split;
        const double bytes = per_sm * kb_part * rows * kMmK;
        double us = std::max(per_sm * kb_part * 1.6 / (C::kStages * ctas), bytes / 130e3);
        us = std::max(us, (double)p.n * p.k / 5e6);
        us = 4.0 + std::max(us, per_sm * epi) + epi;
        if (split > 1) us += 1.6 + 0.01 * NT + 3.0 * (std::ceil(tiles * split / (sms * C::kCtas)) - 1);
        us *= 1.0 + 0.05 * std::min<double>(4.0, tm - 1.0);      // every token tile reads b again
        if (us < best.us) best = {NT, split, us};
    }
}

cudaError_t launch_tc(const SqMatmul& p, int out_type, cudaStream_t st) {
    MmPick pick{0, 1, 1e300};
    const int sms = sm_count();
    mm_estimate<16>(p, sms, pick);
    mm_estimate<32>(p, sms, pick);
    mm_estimate<64>(p, sms, pick);
    mm_estimate<128>(p, sms, pick);
    mm_estimate<256>(p, sms, pick);
    switch (pick.nt) {
        case 16: return go_tc<16>(p, out_type, pick.split, st);
        case 32: return go_tc<32>(p, out_type, pick.split, st);
        case 64: return go_tc<64>(p, out_type, pick.split, st);
        case 128: return go_tc<128>(p, out_type, pick.split, st);
        default: return go_tc<256>(p, out_type, pick.split, st);
    }
}

// one token, or a few whose rows would have to be copied first: dot products
bool use_dot(const SqMatmul& p, bool aligned) { return dot_usable(p) && (p.m == 1 || !aligned); }

// ---- rows that are not 16-byte aligned -------------------------------------
// The tensor copies need aligned rows; others are copied to scratch whose rows
// are, 16 bytes a thread.  Putting the rows together inside the product, by
// warps in the tensor copies' place, took longer (333 x 10007 x 1031: 37 us
// against 17 us; 5000 x 5000 x 5001: 490 us against 127 us).
// Scratch rows are whole 32-byte sectors (333 x 10007 x 1031: 10 us for the product, 13 us with rows of 1040
// bytes) but for short ones, to which that would add a fourth and more.
int64_t mm_ld(int k) { return k <= 64 ? (k + 15) / 16 * 16 : (k + 31) / 32 * 32; }

// Both operands in one launch (blockIdx.y).  A block takes `rows_at_once` rows, about
// 4 chunks a thread: rows are found by one multiplication, from the
// block's first (a division and 64-bit products per chunk took 10.6 us for the
// 10340 rows of 1031 bytes of the first product above).
struct MmAlign {
    const int8_t* rows[2];
    int64_t n[2], ld[2];
    int8_t* to[2];
    int k, chunks;              // 16-byte pieces of a row in scratch
    uint32_t inverse;           // ceil(2^32 / chunks): exact quotients of numbers below 2^19
    int rows_at_once;
};
constexpr int kAlignChunks = 4 * 256;

__global__ void __launch_bounds__(256) mm_align_kernel(const __grid_constant__ MmAlign p) {
    // the product may set itself up meanwhile; it waits for this grid's end before it reads
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int y = blockIdx.y;
    const int64_t n = p.n[y], ld = p.ld[y], last = (n - 1) * ld;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p.rows[y]);
    for (int64_t row0 = (int64_t)blockIdx.x * p.rows_at_once; row0 < n; row0 += (int64_t)gridDim.x * p.rows_at_once) {
        const int64_t first = row0 * ld;
        const int items = (int)min((int64_t)p.rows_at_once, n - row0) * p.chunks;
        uint4* const out = reinterpret_cast<uint4*>(p.to[y]) + row0 * p.chunks;
        for (int t0 = threadIdx.x; t0 < items; t0 += kAlignChunks) {
            SqBytes<false> raw[4];
            uintptr_t at[4];
            int left[4];
            bool inner[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int t = t0 + u * 256;
                const uint32_t r = p.chunks == 1 ? t : __umulhi((uint32_t)t, p.inverse);
                const int c = t - (int)r * p.chunks;
                const int64_t before = first + (int64_t)r * (uint32_t)ld;
                at[u] = lo + before + 16 * c;
                left[u] = t < items ? p.k - 16 * c : 0;          // not above 0: a piece behind the row's end
                inner[u] = before >= 16 && last - before >= 16;  // so many bytes lie before and behind the row
                raw[u].issue_inner(at[u], inner[u] ? left[u] : 0);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (t0 + u * 256 >= items) continue;
                uint4 v = raw[u].take_inner(at[u], left[u]);
                if (!inner[u] && left[u] > 0) v = sq_end_bytes(at[u], at[u] + left[u], lo, lo + last + p.k);
                out[t0 + u * 256] = v;
            }
        }
    }
}

cudaError_t launch_align(MmAlign& p, cudaStream_t st) {
    p.chunks = (int)(mm_ld(p.k) / 16);
    p.inverse = p.chunks == 1 ? 0 : (uint32_t)(((uint64_t(1) << 32) + p.chunks - 1) / p.chunks);
    p.rows_at_once = std::max(1, kAlignChunks / p.chunks);
    const int64_t blocks = (std::max(p.n[0], p.n[1]) + p.rows_at_once - 1) / p.rows_at_once;
    note_launch();
    mm_align_kernel<<<dim3((unsigned)std::min<int64_t>(blocks, (int64_t)sm_count() * 16), p.n[1] ? 2 : 1), 256, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace

size_t sq_matmul_work(const SqMatmul& p) {
    if (p.m == 0 || p.n == 0) return 0;
    const bool al_a = rows_aligned(p.a, p.lda, 16), al_b = rows_aligned(p.b, p.ldb, 16);
    if (use_dot(p, al_a && al_b)) return 0;
    return (size_t)mm_ld(p.k) * ((al_a ? 0 : (size_t)p.m) + (al_b ? 0 : (size_t)p.n));
}

cudaError_t sq_matmul(SqMatmul p, int out_type, void* work, cudaStream_t st) {
    if (p.m == 0 || p.n == 0) return cudaSuccess;
    const bool al_a = rows_aligned(p.a, p.lda, 16), al_b = rows_aligned(p.b, p.ldb, 16);
    if (use_dot(p, al_a && al_b)) {
        MmDot q{};
        q.p = p;
        q.out_type = out_type;
        return launch_dot(q, st);
    }
    if (al_a && al_b) return launch_tc(p, out_type, st);
    MmAlign q{};
    q.k = p.k;
    int8_t* to = static_cast<int8_t*>(work);
    int i = 0;
    auto copied = [&](const int8_t*& rows, int64_t n, int64_t& ld) {
        q.rows[i] = rows;
        q.n[i] = n;
        q.ld[i] = ld;
        q.to[i++] = to;
        rows = to;
        ld = mm_ld(p.k);
        to += n * ld;
    };
    if (!al_b) copied(p.b, p.n, p.ldb);
    if (!al_a) copied(p.a, p.m, p.lda);
    const cudaError_t e = launch_align(q, st);
    return e ? e : launch_tc(p, out_type, st);
}

// Waits for what is queued on st; whether a product on the current device has given up a wait since the last report.
cudaError_t sq_status(bool* gave_up, cudaStream_t st) {
    int seen = 0;
    const int none = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&seen, g_mm_gave_up, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (!e) e = cudaStreamSynchronize(st);
    if (!e && seen) {
        e = cudaMemcpyToSymbolAsync(g_mm_gave_up, &none, sizeof(int), 0, cudaMemcpyHostToDevice, st);
        if (!e) e = cudaStreamSynchronize(st);
    }
    *gave_up = seen != 0;
    return e;
}

// Floating tokens: the dot products quantise them themselves, one launch for
// all.  2 to 4 tokens against much data go to the tensor cores all the same
// (2 x 911870 x 191: 74 us by dot products, whose warps wait for their loads).
static bool fused_scores(const SqMatmul& p) {
    return dot_usable(p) && (p.m == 1 || p.n * p.k <= int64_t(32) << 20 || !rows_aligned(p.b, p.ldb, 16));
}

size_t sq_scores_work(const SqMatmul& q) {
    if (q.m == 0 || q.n == 0 || fused_scores(q)) return 0;
    SqMatmul p = q;
    p.a = nullptr;                                               // the tokens' codes are aligned
    p.lda = mm_ld(p.k);
    return (size_t)p.m * (size_t)(p.lda + 4) + 12 + sq_matmul_work(p);
}

cudaError_t sq_scores(SqWrite w, int x_type, SqMatmul p, int out_type, void* work, cudaStream_t st) {
    if (p.m == 0 || p.n == 0) return cudaSuccess;
    if (fused_scores(p)) {
        MmDot q{};
        q.p = p;
        q.x = w.x;
        q.ldx = w.ldx;
        q.x_type = x_type;
        q.out_type = out_type;
        const int es = x_type == kSqF32 ? 4 : 2;
        q.x_vec = rows_aligned(w.x, (int64_t)w.ldx * es, 16) && (p.k * es) % 16 == 0;
        return launch_dot(q, st);
    }
    // work: the tokens' codes, their scales, then what the product needs
    w.codes = static_cast<uint8_t*>(work);
    w.ldc = (uint32_t)mm_ld(p.k);
    w.scales = reinterpret_cast<float*>(w.codes + (size_t)p.m * w.ldc);
    w.lds = 1;
    w.capacity = w.n;
    const cudaError_t e = sq_write(w, x_type, 8, st);
    if (e) return e;
    p.a = reinterpret_cast<const int8_t*>(w.codes);
    p.a_scale = w.scales;
    p.lda = w.ldc;
    return sq_matmul(p, out_type, w.codes + ((size_t)p.m * (size_t)(w.ldc + 4) + 15) / 16 * 16, st);
}

}  // namespace isb
