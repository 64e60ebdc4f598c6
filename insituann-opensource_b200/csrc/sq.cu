// sq.cu -- scalar-quantised rows: floating rows written to the slots of a store
// as 8-bit or 4-bit codes with one fp32 scale per group of a row, and read
// back.
//
// For a group of values x (the whole row, or `group` consecutive values; the
// last group of a row may be shorter) and L = 127 (8 bits) or 7 (4 bits):
//     scale = fp32(max |x| / L)
//     code  = the whole number nearest to x / scale (ties to even), in [-L, L];
//             0 where the scale is 0
//     value = code * scale in fp32, rounded to the type it is read in.
// The scale is kept in fp32: 4 bytes a group, and an error of 2^-24 next to the
// half step (2^-8 of the group's largest value at 8 bits) that the code costs.
// A group with a NaN or an infinity keeps that NaN or infinity as its scale
// and codes of 0, so it reads back as NaN.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "launch.h"
#include "sq.cuh"

namespace isb {

namespace {

constexpr int kSqThreads = 256;

// Outputs of at least this size are stored evict-first: most of L2 (126 MB)
// stays with the rows that are read, some of them more than once.
constexpr int64_t kSqOnceBytes = int64_t(64) << 20;

constexpr uint32_t kNoSlot = 0xffffffffu;

// slot of a row, kNoSlot outside the store
__device__ __forceinline__ uint32_t sq_slot(const long long* __restrict__ slots, uint32_t row, uint32_t capacity) {
    if (!slots) return row;
    const unsigned long long s = (unsigned long long)slots[row];
    return s < capacity ? (uint32_t)s : kNoSlot;
}

// whether a row after this one has its slot: each of the team's lanes answers
// for its part of the rows
__device__ __forceinline__ bool sq_later(const long long* __restrict__ slots, uint32_t n, uint32_t row, uint32_t slot,
                                         int lane, int team) {
    bool later = false;
    for (uint32_t j = row + 1 + lane; j < n; j += team) later |= slots[j] == (long long)slot;
    return later;
}

// TEAM lanes of a warp take one group, CH chunks each in registers, so a group
// of up to TEAM * CH chunks is read once.  A chunk is 16 bytes of the row (E
// values), or, where rows are not 16-byte aligned or no whole number of chunks,
// one value (two at 4 bits: they share a byte).
template <typename T, int BITS, bool VEC, int TEAM, int CH>
__global__ void __launch_bounds__(kSqThreads, CH <= 4 ? 4 : 2)
    sq_write_kernel(SqWrite p) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    constexpr int TPW = 32 / TEAM;
    const int lane = threadIdx.x & 31, tl = lane % TEAM;
    const uint32_t tmask = TEAM == 32 ? 0xffffffffu : ((1u << (TEAM & 31)) - 1u) << (lane / TEAM * TEAM);
    const uint64_t items = (uint64_t)p.n * (uint32_t)p.groups;
    const uint64_t warp0 = (uint64_t)blockIdx.x * (kSqThreads / 32) + (threadIdx.x >> 5);
    for (uint64_t base = warp0 * TPW; base < items; base += (uint64_t)gridDim.x * (kSqThreads / 32 * TPW)) {
        const uint64_t item = base + lane / TEAM;
        const bool live = item < items;
        uint32_t row = 0;
        int g = 0;
        sq_split(live ? item : 0, p.groups, row, g);
        const int e_lo = g * p.group;
        const int width = live ? min(p.group, p.d - e_lo) : 0;
        const T* xr = static_cast<const T*>(p.x) + (uint64_t)row * p.ldx + e_lo;
        SqRaw<T, E> v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = sq_load<T, VEC, E>(xr, (tl + c * TEAM) * E, width);
        uint32_t slot = live ? sq_slot(p.slots, row, p.capacity) : kNoSlot;
        if (p.dedup == kSqClaim) {
            if (slot != kNoSlot && (uint32_t)p.claim[slot] != row) slot = kNoSlot;
        } else if (p.dedup == kSqScan) {
            const bool later = slot != kNoSlot && sq_later(p.slots, p.n, row, slot, tl, TEAM);
            if (__ballot_sync(0xffffffffu, later) & tmask) slot = kNoSlot;
        }
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c].top(top);
        top = __float_as_uint(sq_top<T>(top));
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (slot == kNoSlot) continue;
        const SqScale s = sq_scale<BITS>(__uint_as_float(top));
        uint8_t* cr = p.codes + (uint64_t)slot * p.ldc + e_lo * BITS / 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (tl + c * TEAM) * E;
            if (e0 < width) sq_store<T, BITS, VEC, E>(cr, e0, width, v[c], s);
        }
        if (tl == 0) p.scales[(uint64_t)slot * p.lds + g] = s.scale;
    }
}

// One block per group, for groups that do not fit a warp's registers: a thread
// keeps its first CH chunks; what a group has beyond kSqThreads * CH is read
// again, from the caches.
template <typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(kSqThreads) sq_write_long_kernel(SqWrite p) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    constexpr int CH = 8;
    __shared__ uint32_t s_top[kSqThreads / 32];
    const uint64_t items = (uint64_t)p.n * (uint32_t)p.groups;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        uint32_t row = 0;
        int g = 0;
        sq_split(item, p.groups, row, g);
        const int e_lo = g * p.group;
        const int width = min(p.group, p.d - e_lo);
        const T* xr = static_cast<const T*>(p.x) + (uint64_t)row * p.ldx + e_lo;
        SqRaw<T, E> v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c] = sq_load<T, VEC, E>(xr, ((int)threadIdx.x + c * kSqThreads) * E, width);
        uint32_t slot = sq_slot(p.slots, row, p.capacity);
        bool later = false;
        if (p.dedup == kSqClaim) {
            if (slot != kNoSlot && (uint32_t)p.claim[slot] != row) slot = kNoSlot;
        } else if (p.dedup == kSqScan && slot != kNoSlot) {
            later = sq_later(p.slots, p.n, row, slot, threadIdx.x, kSqThreads);
        }
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) v[c].top(top);
        for (int e0 = ((int)threadIdx.x + CH * kSqThreads) * E; e0 < width; e0 += kSqThreads * E)
            sq_load<T, VEC, E>(xr, e0, width).top(top);
        top = __reduce_max_sync(0xffffffffu, __float_as_uint(sq_top<T>(top)));
        if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
        if (__syncthreads_or(later)) slot = kNoSlot;
        top = 0;
#pragma unroll
        for (int w = 0; w < kSqThreads / 32; ++w) top = max(top, s_top[w]);
        __syncthreads();                                 // s_top is rewritten by the next group
        if (slot == kNoSlot) continue;                   // the same for the whole block
        const SqScale s = sq_scale<BITS>(__uint_as_float(top));
        uint8_t* cr = p.codes + (uint64_t)slot * p.ldc + e_lo * BITS / 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = ((int)threadIdx.x + c * kSqThreads) * E;
            if (e0 < width) sq_store<T, BITS, VEC, E>(cr, e0, width, v[c], s);
        }
        for (int e0 = ((int)threadIdx.x + CH * kSqThreads) * E; e0 < width; e0 += kSqThreads * E)
            sq_store<T, BITS, VEC, E>(cr, e0, width, sq_load<T, VEC, E>(xr, e0, width), s);
        if (threadIdx.x == 0) p.scales[(uint64_t)slot * p.lds + g] = s.scale;
    }
}

// Which row stays in a slot that several rows name: claim[slot] = the last of
// them.  The table needs no contents of its own: the first kernel leaves one
// row of each named slot there (any of them), the second raises it to the last.
// Where no slot is named twice the second finds its own row and writes nothing.
template <bool RAISE>
__global__ void sq_claim_kernel(const long long* __restrict__ slots, uint32_t n, uint32_t capacity, int* claim) {
    for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) {
        const uint32_t s = sq_slot(slots, i, capacity);
        if (s == kNoSlot) continue;
        if (!RAISE) claim[s] = (int)i;
        else if (*(volatile int*)(claim + s) < (int)i) atomicMax(claim + s, (int)i);
    }
}

// TEAM lanes read a row: lane l takes the chunks l, l + TEAM, ... of 16 bytes of
// output (one value, or two at 4 bits, where the rows are not aligned), CH of
// them at once for each of R rows, so that R * CH loads are in flight.  Row and
// store addresses are found once a row, by shifts: with a division per chunk
// the kernel was bound by its instructions (484 us for 5.12M rows of 128 bf16).
template <typename T, int BITS, bool VEC, int TEAM, int CH, int R>
__global__ void __launch_bounds__(kSqThreads) sq_read_kernel(SqRead p) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
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
                        s[r][c] = scales[r][p.groups == 1 ? 0 : (int)((uint32_t)e0 / (uint32_t)p.group)];
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
                    sq_store_values<T, VEC, E>(out[r], e0, p.d, v, p.once);
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

template <typename T, int BITS, bool VEC, int TEAM, int CH>
cudaError_t go_write(const SqWrite& p, cudaStream_t st) {
    const int64_t per = kSqThreads / TEAM, items = (int64_t)p.n * p.groups;
    const int grid = (int)std::min<int64_t>((items + per - 1) / per, (int64_t)sm_count() * 32);
    note_launch();
    sq_write_kernel<T, BITS, VEC, TEAM, CH><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

// The fewest lanes a group that leave each lane at most 4 chunks (8 for the
// longest groups), so that few shuffles join the maxima and a lane has several
// loads in flight; longer groups take a block.
template <typename T, int BITS, bool VEC>
cudaError_t launch_write(const SqWrite& p, cudaStream_t st) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    const int chunks = (std::min(p.group, p.d) + E - 1) / E;
    if constexpr (VEC) {
        if (chunks <= 2) return go_write<T, BITS, VEC, 2, 1>(p, st);
        if (chunks <= 4) return go_write<T, BITS, VEC, 4, 1>(p, st);
        if (chunks <= 8) return go_write<T, BITS, VEC, 4, 2>(p, st);
        if (chunks <= 12) return go_write<T, BITS, VEC, 4, 3>(p, st);
        if (chunks > 16 && chunks <= 24) return go_write<T, BITS, VEC, 8, 3>(p, st);
        if (chunks > 16 && chunks <= 32) return go_write<T, BITS, VEC, 8, 4>(p, st);
        if (chunks > 64 && chunks <= 128) return go_write<T, BITS, VEC, 32, 4>(p, st);
    }
    if (chunks <= 16) return go_write<T, BITS, VEC, 4, 4>(p, st);
    if (chunks <= 64) return go_write<T, BITS, VEC, 16, 4>(p, st);
    if (chunks <= 256) return go_write<T, BITS, VEC, 32, 8>(p, st);
    const int grid = (int)std::min<int64_t>((int64_t)p.n * p.groups, (int64_t)sm_count() * 8);
    note_launch();
    sq_write_long_kernel<T, BITS, VEC><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

template <typename T, int BITS, bool VEC, int TEAM, int CH, int R>
cudaError_t go_read(const SqRead& p, cudaStream_t st) {
    const int64_t per = kSqThreads / TEAM * R;
    const int grid = (int)std::min<int64_t>(((int64_t)p.n + per - 1) / per, (int64_t)sm_count() * 64);
    note_launch();
    sq_read_kernel<T, BITS, VEC, TEAM, CH, R><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

// A lane takes up to 4 chunks of a row (so that a row's addresses are found once
// for them) of up to 4 rows; a row that is no multiple of the lanes leaves the fewest idle.
template <typename T, int BITS, bool VEC>
cudaError_t launch_read(const SqRead& p, cudaStream_t st) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    const int chunks = (p.d + E - 1) / E;
    if constexpr (VEC) {
        if (chunks <= 2) return go_read<T, BITS, VEC, 2, 1, 4>(p, st);
        if (chunks > 4 && chunks <= 8) return go_read<T, BITS, VEC, 4, 2, 2>(p, st);
        if (chunks > 8 && chunks <= 12) return go_read<T, BITS, VEC, 4, 3, 2>(p, st);
        if (chunks > 16 && chunks <= 24) return go_read<T, BITS, VEC, 8, 3, 2>(p, st);
        if (chunks > 24 && chunks <= 32) return go_read<T, BITS, VEC, 8, 4, 2>(p, st);
    }
    if (chunks <= 4) return go_read<T, BITS, VEC, 4, 1, 4>(p, st);
    if (chunks <= 16) return go_read<T, BITS, VEC, 4, 4, 2>(p, st);
    return go_read<T, BITS, VEC, 32, 4, 1>(p, st);
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

cudaError_t sq_write(SqWrite p, int type, int bits, cudaStream_t st) {
    if (p.n == 0) return cudaSuccess;
    p.groups = p.group ? (p.d + p.group - 1) / p.group : 1;
    if (!p.group) p.group = p.d;
    p.dedup = !p.slots || p.n == 1 ? kSqAll : p.n <= kSqScanRows ? kSqScan : kSqClaim;
    if (p.dedup == kSqClaim) {
        const int grid = (int)std::min<int64_t>(((int64_t)p.n + 255) / 256, (int64_t)sm_count() * 16);
        note_launch(2);
        sq_claim_kernel<false><<<grid, 256, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
        sq_claim_kernel<true><<<grid, 256, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
        const cudaError_t e = cudaGetLastError();
        if (e) return e;
    }
    const int es = type == kSqF32 ? 4 : 2;
    // a 16-byte chunk of values makes 4 or 8 (8 bits), 2 or 4 (4 bits) bytes of codes
    const size_t cw = (size_t)(16 / es) * bits / 8;
    const bool vec = aligned(p.x, 16) && ((int64_t)p.ldx * es) % 16 == 0 && (p.d * es) % 16 == 0 &&
                     aligned(p.codes, cw) && p.ldc % cw == 0;
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        if (bits == 8) return vec ? launch_write<T, 8, true>(p, st) : launch_write<T, 8, false>(p, st);
        return vec ? launch_write<T, 4, true>(p, st) : launch_write<T, 4, false>(p, st);
    });
}

cudaError_t sq_read(SqRead p, int type, int bits, cudaStream_t st) {
    if (p.n == 0) return cudaSuccess;
    p.groups = p.group ? (p.d + p.group - 1) / p.group : 1;
    if (!p.group) p.group = p.d;
    const int es = type == kSqF32 ? 4 : 2;
    const size_t cw = (size_t)(16 / es) * bits / 8;
    const bool vec = aligned(p.out, 16) && ((int64_t)p.ldo * es) % 16 == 0 && (p.d * es) % 16 == 0 &&
                     aligned(p.codes, cw) && p.ldc % cw == 0;
    p.once = (int64_t)p.n * p.d * es >= kSqOnceBytes;
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        if (bits == 8) return vec ? launch_read<T, 8, true>(p, st) : launch_read<T, 8, false>(p, st);
        return vec ? launch_read<T, 4, true>(p, st) : launch_read<T, 4, false>(p, st);
    });
}

}  // namespace isb
