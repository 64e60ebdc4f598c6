// sq_mm.cu -- 8-bit matrix product with a scale per token and per channel:
//     out[i, j] = float(sum_t a[i, t] * b[j, t]) * a_scale[i] * b_scale[j] + bias[j]
// a [m, k] and b [n, k] int8, both with k innermost.  The sum is exact in 32
// bits (k < 2^17); the scaling and the bias are fp32 and each output is
// rounded once more, to its type.
#include <algorithm>

#include "launch.h"
#include "sq.cuh"

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

bool rows_aligned(const void* p, int64_t ld, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0 && ld % a == 0; }

template <typename T>
cudaError_t launch_mm(const SqMatmul& p, cudaStream_t st) {
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
