// sq.cu -- scalar-quantised rows: floating rows written to the slots of a store
// as 8-bit or 4-bit codes with one fp32 scale per group of a row, and read
// back.
//
// For a group of values x (the whole row, or `group` consecutive values; the
// last group of a row may be shorter) and L = 127 (8 bits) or 7 (4 bits):
//     scale = fp32(max |x| / L)
//     code  = the whole number nearest to x / scale (ties to even), in [-L, L];
//             0 where the scale is 0
//     value = code * scale, rounded once to the type it is read in.
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

// slot of row r, or -1 where the row is not written: slots outside the store,
// and rows whose slot a later row names too.  The lanes `lane` of a team of
// `team` threads share the search; every lane gets its own part's answer
// (`later`), which the caller combines.
__device__ __forceinline__ bool sq_later_same_slot(const long long* __restrict__ slots, int64_t n, int64_t row,
                                                   long long slot, int lane, int team) {
    bool later = false;
    for (int64_t j = row + 1 + lane; j < n; j += team) later |= slots[j] == slot;
    return later;
}

// TEAM lanes of a warp take one group, CH chunks each in registers, so a group
// of up to TEAM * CH chunks is read once.  A chunk is 16 bytes of the row (E
// values), or, where rows are not 16-byte aligned, one value (two at 4 bits:
// they share a byte).
template <typename T, int BITS, bool VEC, int TEAM, int CH>
__global__ void __launch_bounds__(kSqThreads)
    sq_write_kernel(SqWrite p) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    constexpr int TPW = 32 / TEAM;
    const int lane = threadIdx.x & 31, tl = lane % TEAM;
    const uint32_t tmask = TEAM == 32 ? 0xffffffffu : ((1u << (TEAM & 31)) - 1u) << (lane / TEAM * TEAM);
    const int64_t items = p.n * p.groups;
    const int64_t warp0 = (int64_t)blockIdx.x * (kSqThreads / 32) + (threadIdx.x >> 5);
    for (int64_t base = warp0 * TPW; base < items; base += (int64_t)gridDim.x * (kSqThreads / 32) * TPW) {
        const int64_t item = base + lane / TEAM;
        bool live = item < items;
        int64_t row = 0;
        int g = 0;
        sq_split(live ? item : 0, p.groups, row, g);
        const int e_lo = g * p.group;
        const int width = min(p.group, p.d - e_lo);
        const T* xr = static_cast<const T*>(p.x) + row * p.ldx + e_lo;
        float v[CH][E];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (tl + c * TEAM) * E;
            sq_load<T, VEC, E>(xr, e0, live ? width : 0, v[c]);
        }
        int64_t slot = -1;
        if (live) {
            slot = p.slots ? p.slots[row] : row;
            if (slot < 0 || slot >= p.capacity) slot = -1;
            if (slot >= 0 && p.dedup == kSqClaim && p.claim[slot] != (int)row) slot = -1;
        }
        if (p.dedup == kSqScan) {
            const bool later = slot >= 0 && sq_later_same_slot(p.slots, p.n, row, slot, tl, TEAM);
            if (__ballot_sync(0xffffffffu, later) & tmask) slot = -1;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(v[c][e]) & 0x7fffffffu);
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (slot < 0) continue;
        const SqScale s = sq_scale<BITS>(top);
        uint8_t* cr = p.codes + slot * p.ldc + e_lo * BITS / 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (tl + c * TEAM) * E;
            if (e0 < width) sq_store<BITS, VEC, E>(cr, e0, width, v[c], s);
        }
        if (tl == 0) p.scales[slot * p.lds + g] = s.scale;
    }
}

// One block per group, for groups that do not fit a warp's registers: the group
// is read twice, the second time from the caches.
template <typename T, int BITS, bool VEC>
__global__ void __launch_bounds__(kSqThreads) sq_write_long_kernel(SqWrite p) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    __shared__ uint32_t s_top[kSqThreads / 32];
    const int64_t items = p.n * p.groups;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        int64_t row = 0;
        int g = 0;
        sq_split(item, p.groups, row, g);
        int64_t slot = p.slots ? p.slots[row] : row;
        if (slot < 0 || slot >= p.capacity) slot = -1;
        if (slot >= 0 && p.dedup == kSqClaim && p.claim[slot] != (int)row) slot = -1;
        bool later = false;
        if (p.dedup == kSqScan && slot >= 0)
            later = sq_later_same_slot(p.slots, p.n, row, slot, threadIdx.x, kSqThreads);
        if (__syncthreads_or(later)) slot = -1;
        if (slot < 0) continue;                          // the same for the whole block
        const int e_lo = g * p.group;
        const int width = min(p.group, p.d - e_lo);
        const T* xr = static_cast<const T*>(p.x) + row * p.ldx + e_lo;
        uint32_t top = 0;
        for (int e0 = threadIdx.x * E; e0 < width; e0 += kSqThreads * E) {
            float v[E];
            sq_load<T, VEC, E>(xr, e0, width, v);
#pragma unroll
            for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
        __syncthreads();
        top = 0;
#pragma unroll
        for (int w = 0; w < kSqThreads / 32; ++w) top = max(top, s_top[w]);
        const SqScale s = sq_scale<BITS>(top);
        uint8_t* cr = p.codes + slot * p.ldc + e_lo * BITS / 8;
        for (int e0 = threadIdx.x * E; e0 < width; e0 += kSqThreads * E) {
            float v[E];
            sq_load<T, VEC, E>(xr, e0, width, v);
            sq_store<BITS, VEC, E>(cr, e0, width, v, s);
        }
        if (threadIdx.x == 0) p.scales[slot * p.lds + g] = s.scale;
        __syncthreads();                                 // s_top is rewritten by the next group
    }
}

// Which row stays in a slot that several rows name: claim[slot] = the last of
// them.  The table needs no contents of its own: the first kernel clears what
// the second one raises.
__global__ void sq_claim_clear_kernel(const long long* __restrict__ slots, int64_t n, int64_t capacity,
                                      int* __restrict__ claim) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const long long s = slots[i];
        if (s >= 0 && s < capacity) claim[s] = -1;
    }
}

__global__ void sq_claim_kernel(const long long* __restrict__ slots, int64_t n, int64_t capacity,
                                int* __restrict__ claim) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const long long s = slots[i];
        if (s >= 0 && s < capacity) atomicMax(claim + s, (int)i);
    }
}

// A thread per chunk of a row's values: 16 bytes of output, or one value (two
// at 4 bits) where the rows are not aligned.  U chunks per thread are in flight.
template <typename T, int BITS, bool VEC, int U>
__global__ void __launch_bounds__(kSqThreads) sq_read_kernel(SqRead p) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    constexpr int W = E * BITS / 8 > 0 ? E * BITS / 8 : 1;       // bytes of codes per chunk
    const int cpr = (p.d + E - 1) / E;
    const int64_t items = p.n * cpr;
    for (int64_t b0 = (int64_t)blockIdx.x * (kSqThreads * U); b0 < items;
         b0 += (int64_t)gridDim.x * (kSqThreads * U)) {
        int64_t row[U], slot[U];
        int e0[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t item = b0 + u * kSqThreads + threadIdx.x;
            int c = 0;
            row[u] = -1;
            slot[u] = -1;
            e0[u] = 0;
            if (item < items) {
                sq_split(item, cpr, row[u], c);
                e0[u] = c * E;
                slot[u] = p.slots ? p.slots[row[u]] : row[u];
                if (slot[u] < 0 || slot[u] >= p.capacity) slot[u] = -1;
            }
        }
        uint8_t q[U][W];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) q[u][w] = 0;
            if (slot[u] >= 0) {
                sq_load_codes<VEC, W>(p.codes + slot[u] * p.ldc, e0[u] * BITS / 8, (p.d * BITS + 7) / 8, q[u]);
                s[u] = p.scales[slot[u] * p.lds + (p.groups == 1 ? 0 : e0[u] / p.group)];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row[u] < 0) continue;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (float)sq_code<BITS>(q[u], e) * s[u];
            sq_store_values<T, VEC, E>(static_cast<T*>(p.out) + row[u] * p.ldo, e0[u], p.d, v);
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

template <typename T, int BITS, bool VEC>
cudaError_t launch_write(const SqWrite& p, cudaStream_t st) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    const int64_t items = p.n * p.groups;
    const int64_t chunks = (std::min(p.group, p.d) + E - 1) / E;
    const int sms = sm_count();
    note_launch();
    // 8 lanes x 4 chunks: 512 bytes of row per 8 lanes (a warp reads 4 rows'
    // lines at once); 32 lanes x 8 chunks: 4 KB; longer groups take a block
    if (chunks <= 8 * 4) {
        const int64_t per = kSqThreads / 8;
        const int grid = (int)std::min<int64_t>((items + per - 1) / per, (int64_t)sms * 32);
        sq_write_kernel<T, BITS, VEC, 8, 4><<<grid, kSqThreads, 0, st>>>(p);
    } else if (chunks <= 32 * 8) {
        const int64_t per = kSqThreads / 32;
        const int grid = (int)std::min<int64_t>((items + per - 1) / per, (int64_t)sms * 32);
        sq_write_kernel<T, BITS, VEC, 32, 8><<<grid, kSqThreads, 0, st>>>(p);
    } else {
        const int grid = (int)std::min<int64_t>(items, (int64_t)sms * 8);
        sq_write_long_kernel<T, BITS, VEC><<<grid, kSqThreads, 0, st>>>(p);
    }
    return cudaGetLastError();
}

template <typename T, int BITS, bool VEC>
cudaError_t launch_read(const SqRead& p, cudaStream_t st) {
    constexpr int E = sq_chunk<T, BITS, VEC>();
    constexpr int U = 4;
    const int64_t items = p.n * ((p.d + E - 1) / E);
    const int64_t per = kSqThreads * U;
    const int grid = (int)std::min<int64_t>((items + per - 1) / per, (int64_t)sm_count() * 64);
    note_launch();
    sq_read_kernel<T, BITS, VEC, U><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace

cudaError_t sq_write(SqWrite p, int type, int bits, cudaStream_t st) {
    if (p.n == 0) return cudaSuccess;
    p.groups = p.group ? (p.d + p.group - 1) / p.group : 1;
    if (!p.group) p.group = p.d;
    p.dedup = !p.slots || p.n == 1 ? kSqAll : p.n <= kSqScanRows ? kSqScan : kSqClaim;
    if (p.dedup == kSqClaim) {
        const int grid = (int)std::min<int64_t>((p.n + 255) / 256, (int64_t)sm_count() * 16);
        note_launch(2);
        sq_claim_clear_kernel<<<grid, 256, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
        sq_claim_kernel<<<grid, 256, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
        const cudaError_t e = cudaGetLastError();
        if (e) return e;
    }
    const int es = type == kSqF32 ? 4 : 2;
    // a 16-byte chunk of values makes 4 or 8 (8 bits), 2 or 4 (4 bits) bytes of codes
    const size_t cw = (size_t)(16 / es) * bits / 8;
    const bool vec = aligned(p.x, 16) && (p.ldx * es) % 16 == 0 && aligned(p.codes, cw) && p.ldc % cw == 0;
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
    const bool vec = aligned(p.out, 16) && (p.ldo * es) % 16 == 0 && aligned(p.codes, cw) && p.ldc % cw == 0;
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        if (bits == 8) return vec ? launch_read<T, 8, true>(p, st) : launch_read<T, 8, false>(p, st);
        return vec ? launch_read<T, 4, true>(p, st) : launch_read<T, 4, false>(p, st);
    });
}

}  // namespace isb
