// sq_read.cu -- scalar-quantised rows read back: the values of a list of slots.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "launch.h"
#include "sq.cuh"

namespace isb {

namespace {

constexpr int kSqThreads = 256;

// Outputs of at least this size are stored evict-first: most of L2 (126 MB)
// stays with the rows that are read, some of them more than once.
constexpr int64_t kSqOnceBytes = int64_t(64) << 20;

// the group of a row's value e
__device__ __forceinline__ int sq_group(const SqRead& p, int e) {
    return p.groups == 1 ? 0 : p.group_log >= 0 ? e >> p.group_log : (int)((uint32_t)e / (uint32_t)p.group);
}

// TEAM lanes read a row: lane l takes the chunks l, l + TEAM, ... of 16 bytes of
// output (one value, or two at 4 bits, where the rows are not aligned), CH of
// them at once for each of R rows, so that R * CH loads are in flight.  Row and
// store addresses are found once a row, by shifts: with a division per chunk
// the kernel was bound by its instructions (484 us for 5.12M rows of 128 bf16).
template <typename T, int BITS, int MODE, int TEAM, int CH, int R>
__global__ void __launch_bounds__(kSqThreads) sq_read_kernel(SqRead p) {
    constexpr int E = sq_chunk<T, BITS, MODE>();
    constexpr int W = E * BITS / 8;                              // bytes of codes per chunk
    constexpr int TPB = kSqThreads / TEAM;
    const int tl = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    for (uint32_t r0 = blockIdx.x * (TPB * R); r0 < p.n; r0 += gridDim.x * (TPB * R)) {
        uint32_t slot[R];
        const uint8_t* codes[R];
        const float* scales[R];
        T* out[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t row = r0 + r * TPB + team;
            const bool live = row < p.n;
            slot[r] = live ? sq_slot(p.slots, row, p.capacity) : kNoSlot;
            out[r] = live ? static_cast<T*>(p.out) + (uint64_t)row * p.ldo : nullptr;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            codes[r] = p.codes + (uint64_t)slot[r] * p.ldc;
            scales[r] = p.scales + (uint64_t)slot[r] * p.lds;
        }
        for (int e1 = tl * E; e1 < p.d; e1 += TEAM * CH * E) {
            uint32_t q[R][CH][(W + 3) / 4];
            float s[R][CH];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int e0 = e1 + c * TEAM * E;
                    if (slot[r] != kNoSlot && e0 < p.d) {
                        sq_load_codes<W>(codes[r] + e0 * BITS / 8, q[r][c]);
                        s[r][c] = scales[r][sq_group(p, e0)];
                    } else {
#pragma unroll
                        for (int w = 0; w < (W + 3) / 4; ++w) q[r][c][w] = 0;
                        s[r][c] = 0.f;
                    }
                }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int e0 = e1 + c * TEAM * E;
                    if (!out[r] || e0 >= p.d) continue;
                    float v[E];
                    sq_values<BITS, E>(q[r][c], s[r][c], v);
                    sq_store_values<T, MODE == kSqVec, E>(out[r], e0, p.d, v, p.once);
                }
        }
    }
}

// the last word of a store's last row, of which `n` bytes are there
__device__ __noinline__ uint32_t sq_last_word(const uint8_t* at, int n) {
    uint32_t w = 0;
    for (int k = 0; k < n && k < 4; ++k) w |= (uint32_t)at[k] << (8 * k);
    return w;
}

// The same for output rows that are not aligned (an odd d, a slice): chunks are
// 16 aligned bytes of output, so a row's first and last chunk may be a part (stored value by
// value) and a chunk's codes start anywhere, at a nibble too: they are shifted
// out of aligned words.  459587 rows of 90 fp16 in 48 us, 100 us value by value throughout
// (floor 20 us).
template <typename T, int BITS, int TEAM, int CH, int R>
__global__ void __launch_bounds__(kSqThreads) sq_read_shifted_kernel(SqRead p) {
    constexpr int E = 16 / (int)sizeof(T);
    constexpr int NW = (E * BITS + 31) / 32;                     // words of a chunk's codes once shifted
    constexpr int TPB = kSqThreads / TEAM;
    const int tl = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const int bytes = (p.d * BITS + 7) / 8;
    for (uint32_t r0 = blockIdx.x * (TPB * R); r0 < p.n; r0 += gridDim.x * (TPB * R)) {
        uint32_t slot[R];
        const uint8_t* codes[R];
        const float* scales[R];
        T* out[R];
        int past[R];                                             // values from an aligned address to the row
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t row = r0 + r * TPB + team;
            const bool live = row < p.n;
            slot[r] = live ? sq_slot(p.slots, row, p.capacity) : kNoSlot;
            out[r] = live ? static_cast<T*>(p.out) + (uint64_t)row * p.ldo : nullptr;
            past[r] = (int)(reinterpret_cast<uintptr_t>(out[r]) & 15) / (int)sizeof(T);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            codes[r] = p.codes + (uint64_t)slot[r] * p.ldc;
            scales[r] = p.scales + (uint64_t)slot[r] * p.lds;
        }
        for (int e1 = tl * E; e1 < p.d + E; e1 += TEAM * CH * E) {
            uint32_t w[R][CH][NW + 1];
            float s0[R][CH], s1[R][CH];
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int e0 = e1 + c * TEAM * E - past[r], w0 = (e0 * BITS) >> 5;
                    const bool get = slot[r] != kNoSlot && e0 < p.d;
#pragma unroll
                    for (int i = 0; i <= NW; ++i) {
                        const int b = (w0 + i) * 4;              // the word's first byte of the row
                        w[r][c][i] = 0;
                        if (get && b >= 0 && b < bytes) {
                            // the store may end inside its last row's last word
                            if (b + 4 <= bytes || slot[r] + 1 < p.capacity)
                                w[r][c][i] = *reinterpret_cast<const uint32_t*>(codes[r] + b);
                            else w[r][c][i] = sq_last_word(codes[r] + b, bytes - b);
                        }
                    }
                    s0[r][c] = s1[r][c] = 0.f;
                    if (get) {
                        s0[r][c] = scales[r][sq_group(p, max(e0, 0))];
                        s1[r][c] = p.groups == 1 ? s0[r][c] : scales[r][sq_group(p, min(e0 + E, p.d) - 1)];
                    }
                }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const int e0 = e1 + c * TEAM * E - past[r];
                    if (!out[r] || e0 >= p.d) continue;
                    uint32_t q[NW];
#pragma unroll
                    for (int i = 0; i < NW; ++i)
                        q[i] = __funnelshift_r(w[r][c][i], w[r][c][i + 1], (uint32_t)(e0 * BITS) & 31u);
                    float v[E];
                    if (p.groups == 1) sq_values<BITS, E>(q, s0[r][c], v);
                    else {
                        sq_values<BITS, E>(q, 1.f, v);           // the codes themselves
                        // a chunk meets two groups at most: the second starts at a multiple of 16 values
                        const int turn = sq_group(p, min(e0 + E, p.d) - 1) * p.group - e0;
#pragma unroll
                        for (int e = 0; e < E; ++e) v[e] *= e >= turn ? s1[r][c] : s0[r][c];
                    }
                    if (e0 >= 0 && e0 + E <= p.d) sq_store_values<T, true, E>(out[r], e0, p.d, v, p.once);
                    else {
#pragma unroll
                        for (int e = 0; e < E; ++e)
                            if (e0 + e >= 0 && e0 + e < p.d) sq_round(v[e], out[r][e0 + e]);
                    }
                }
        }
    }
}

int sm_count() {
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

template <typename F>
cudaError_t by_type(int type, F&& f) {
    if (type == kSqF32) return f(float{});
    if (type == kSqF16) return f(__half{});
    return f(__nv_bfloat16{});
}

template <typename T, int BITS, int MODE, int TEAM, int CH, int R>
cudaError_t go_read(const SqRead& p, cudaStream_t st) {
    const int64_t per = kSqThreads / TEAM * R;
    const int grid = (int)std::min<int64_t>(((int64_t)p.n + per - 1) / per, (int64_t)sm_count() * 64);
    note_launch();
    sq_read_kernel<T, BITS, MODE, TEAM, CH, R><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

// A lane takes up to 4 chunks of a row (so that a row's addresses are found once
// for them) of up to 4 rows; a row that is no multiple of the lanes leaves the fewest idle.
template <typename T, int BITS, int MODE>
cudaError_t launch_read(const SqRead& p, cudaStream_t st) {
    constexpr int E = sq_chunk<T, BITS, MODE>();
    const int chunks = (p.d + E - 1) / E;
    if constexpr (MODE == kSqVec) {
        if (chunks <= 2) return go_read<T, BITS, MODE, 2, 1, 4>(p, st);
        if (chunks > 4 && chunks <= 8) return go_read<T, BITS, MODE, 4, 2, 2>(p, st);
        if (chunks > 8 && chunks <= 12) return go_read<T, BITS, MODE, 4, 3, 2>(p, st);
        if (chunks > 16 && chunks <= 24) return go_read<T, BITS, MODE, 8, 3, 2>(p, st);
        if (chunks > 24 && chunks <= 32) return go_read<T, BITS, MODE, 8, 4, 2>(p, st);
        if (chunks > 4 && chunks <= 16) return go_read<T, BITS, MODE, 4, 4, 2>(p, st);
        if (chunks > 32 && chunks <= 64) return go_read<T, BITS, MODE, 16, 4, 1>(p, st);
    } else {
        // neighbouring lanes store neighbouring values
        if (chunks > 4 && chunks <= 8) return go_read<T, BITS, MODE, 8, 1, 4>(p, st);
        if (chunks > 8 && chunks <= 16) return go_read<T, BITS, MODE, 16, 1, 4>(p, st);
        if (chunks > 16 && chunks <= 32) return go_read<T, BITS, MODE, 32, 1, 4>(p, st);
        if (chunks > 32 && chunks <= 64) return go_read<T, BITS, MODE, 32, 2, 2>(p, st);
    }
    if (chunks <= 4) return go_read<T, BITS, MODE, 4, 1, 4>(p, st);
    return go_read<T, BITS, MODE, 32, 4, 1>(p, st);
}

template <typename T, int BITS, int TEAM, int CH, int R>
cudaError_t go_shifted(const SqRead& p, cudaStream_t st) {
    const int64_t per = kSqThreads / TEAM * R;
    const int grid = (int)std::min<int64_t>(((int64_t)p.n + per - 1) / per, (int64_t)sm_count() * 64);
    note_launch();
    sq_read_shifted_kernel<T, BITS, TEAM, CH, R><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int BITS>
cudaError_t launch_shifted(const SqRead& p, cudaStream_t st) {
    const int chunks = p.d / (16 / (int)sizeof(T)) + 2;          // at most
    if (chunks <= 4) return go_shifted<T, BITS, 4, 1, 4>(p, st);
    if (chunks <= 8) return go_shifted<T, BITS, 4, 2, 2>(p, st);
    if (chunks <= 16) return go_shifted<T, BITS, 8, 2, 2>(p, st);
    if (chunks <= 64) return go_shifted<T, BITS, 16, 2, 2>(p, st);
    if (chunks <= 128) return go_shifted<T, BITS, 32, 2, 2>(p, st);
    return go_shifted<T, BITS, 32, 4, 1>(p, st);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

cudaError_t sq_read(SqRead p, int type, int bits, cudaStream_t st) {
    if (p.n == 0) return cudaSuccess;
    p.groups = p.group ? (p.d + p.group - 1) / p.group : 1;
    if (!p.group) p.group = p.d;
    const int es = type == kSqF32 ? 4 : 2;
    const size_t cw = (size_t)(16 / es) * bits / 8;
    const bool vec = aligned(p.out, 16) && ((int64_t)p.ldo * es) % 16 == 0 && (p.d * es) % 16 == 0 &&
                     aligned(p.codes, cw) && p.ldc % cw == 0;
    p.once = (int64_t)p.n * p.d * es >= kSqOnceBytes;
    p.group_log = (p.group & (p.group - 1)) == 0 ? 31 - __builtin_clz((unsigned)p.group) : -1;
    // rows of less than two chunks are mostly ends: value by value
    const bool words = aligned(p.codes, 4) && p.ldc % 4 == 0 && p.d * es >= 32;
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        if (bits == 8)
            return vec ? launch_read<T, 8, kSqVec>(p, st)
                       : words ? launch_shifted<T, 8>(p, st) : launch_read<T, 8, kSqSingle>(p, st);
        return vec ? launch_read<T, 4, kSqVec>(p, st)
                   : words ? launch_shifted<T, 4>(p, st) : launch_read<T, 4, kSqSingle>(p, st);
    });
}

}  // namespace isb
