// sq_write.cu -- floating rows written to the slots of a store of scalar-quantised
// rows: 8-bit or 4-bit codes with one fp32 scale per group of a row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "launch.h"
#include "sq.cuh"

namespace isb {

namespace {

constexpr int kSqThreads = 256;

// whether a row after this one has its slot: each of the team's lanes answers
// for its part of the rows
__device__ __forceinline__ bool sq_later(const long long* __restrict__ slots, uint32_t n, uint32_t row, uint32_t slot,
                                         int lane, int team) {
    bool later = false;
#pragma unroll 4
    for (uint32_t j = row + 1 + lane; j < n; j += team) later |= slots[j] == (long long)slot;
    return later;
}

// TEAM lanes of a warp take one group, CH chunks each in registers, so a group
// of up to TEAM * CH chunks (E values each, sq_chunk) is read once.
template <typename T, int BITS, int MODE, int TEAM, int CH>
__global__ void __launch_bounds__(kSqThreads, CH > 4 ? 2 : MODE == kSqShifted && CH > 2 ? 3 : 4)
    sq_write_kernel(SqWrite p) {
    // a product queued behind may set itself up; it waits for this grid's end before it reads
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int E = sq_chunk<T, BITS, MODE>();
    constexpr int TPW = 32 / TEAM;
    const int lane = threadIdx.x & 31, tl = lane % TEAM;
    const uint32_t tmask = (TEAM == 32 ? 0xffffffffu : (1u << (TEAM & 31)) - 1u) << (lane / TEAM * TEAM);
    SqSpan span;
    span.lo = reinterpret_cast<uintptr_t>(p.x);
    span.hi = span.lo + ((uint64_t)(p.n - 1) * p.ldx + p.d) * sizeof(T);
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
        span.at(xr, width);
        SqLoad<T, MODE, E> in[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) in[c].issue(xr, (tl + c * TEAM) * E, width, span);
        uint32_t slot = live ? sq_slot(p.slots, row, p.capacity) : kNoSlot;
        if (p.dedup == kSqClaim) {
            if (slot != kNoSlot && (uint32_t)p.claim[slot] != row) slot = kNoSlot;
        } else if (p.dedup == kSqScan) {
            const bool later = slot != kNoSlot && sq_later(p.slots, p.n, row, slot, tl, TEAM);
            if (__ballot_sync(0xffffffffu, later) & tmask) slot = kNoSlot;
        }
        uint32_t top = 0;
        SqRaw<T, E> v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (MODE == kSqShifted && c * TEAM * E >= width) break;
            v[c] = in[c].take(xr, (tl + c * TEAM) * E, width, span);
            v[c].top(top);
        }
        top = __float_as_uint(sq_top<T>(top));
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (slot == kNoSlot) continue;
        const SqScale s = sq_scale<BITS>(__uint_as_float(top));
        uint8_t* cr = p.codes + (uint64_t)slot * p.ldc + e_lo * BITS / 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (tl + c * TEAM) * E;
            if (e0 < width) sq_store<T, BITS, MODE, E>(cr, e0, width, v[c], s);
        }
        if (tl == 0) p.scales[(uint64_t)slot * p.lds + g] = s.scale;
    }
}

// One block per group, for groups that do not fit a warp's registers: a thread
// keeps its first CH chunks; what a group has beyond kSqThreads * CH is read
// again, from the caches.
template <typename T, int BITS, int MODE, int CH>
__global__ void __launch_bounds__(kSqThreads, CH <= 2 ? 4 : MODE == kSqShifted ? CH <= 4 ? 2 : 1 : 3) sq_write_long_kernel(SqWrite p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // as above
    constexpr int E = sq_chunk<T, BITS, MODE>();
    __shared__ uint32_t s_top[kSqThreads / 32];
    SqSpan span;
    span.lo = reinterpret_cast<uintptr_t>(p.x);
    span.hi = span.lo + ((uint64_t)(p.n - 1) * p.ldx + p.d) * sizeof(T);
    const uint64_t items = (uint64_t)p.n * (uint32_t)p.groups;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        uint32_t row = 0;
        int g = 0;
        sq_split(item, p.groups, row, g);
        const int e_lo = g * p.group;
        const int width = min(p.group, p.d - e_lo);
        const T* xr = static_cast<const T*>(p.x) + (uint64_t)row * p.ldx + e_lo;
        span.at(xr, width);
        SqLoad<T, MODE, E> in[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (MODE == kSqVec || c * kSqThreads * E < width) in[c].issue(xr, ((int)threadIdx.x + c * kSqThreads) * E, width, span);
        uint32_t slot = sq_slot(p.slots, row, p.capacity);
        bool later = false;
        if (p.dedup == kSqClaim) {
            if (slot != kNoSlot && (uint32_t)p.claim[slot] != row) slot = kNoSlot;
        } else if (p.dedup == kSqScan && slot != kNoSlot) {
            later = sq_later(p.slots, p.n, row, slot, threadIdx.x, kSqThreads);
        }
        uint32_t top = 0;
        SqRaw<T, E> v[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (MODE != kSqVec && c * kSqThreads * E >= width) break;
            v[c] = in[c].take(xr, ((int)threadIdx.x + c * kSqThreads) * E, width, span);
            v[c].top(top);
        }
        for (int e0 = ((int)threadIdx.x + CH * kSqThreads) * E; e0 < width; e0 += kSqThreads * E) {
            SqLoad<T, MODE, E> more;
            more.issue(xr, e0, width, span);
            more.take(xr, e0, width, span).top(top);
        }
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
            if (e0 < width) sq_store<T, BITS, MODE, E>(cr, e0, width, v[c], s);
        }
        for (int e0 = ((int)threadIdx.x + CH * kSqThreads) * E; e0 < width; e0 += kSqThreads * E) {
            SqLoad<T, MODE, E> more;
            more.issue(xr, e0, width, span);
            sq_store<T, BITS, MODE, E>(cr, e0, width, more.take(xr, e0, width, span), s);
        }
        if (threadIdx.x == 0) p.scales[(uint64_t)slot * p.lds + g] = s.scale;
    }
}

// Which row stays in a slot that several rows name: claim[slot] = the last of
// them.  The table needs no contents of its own: the first pass leaves one row
// of each named slot there (any of them), the second raises it to the last.
// Where no slot is named twice the second finds its own row and writes nothing.
// Up to kClaimRows rows one cluster runs both passes, with its barrier between
// them: a launch less (2.3 us of the host; the GPU itself takes 0.8 us longer at
// 4099 rows, 1.8 us at 10000); more rows need more SMs.
constexpr uint32_t kClaimRows = 16384;
constexpr int kClaimCtas = 8, kClaimThreads = 1024;

template <bool RAISE>
__device__ __forceinline__ void sq_claim_pass(const long long* __restrict__ slots, uint32_t n, uint32_t capacity,
                                              int* claim) {
    const uint32_t step = gridDim.x * blockDim.x;
    for (uint32_t i0 = blockIdx.x * blockDim.x + threadIdx.x; i0 < n; i0 += 4 * step) {
        uint32_t s[4];
        int c[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = i0 + u * step < n ? sq_slot(slots, i0 + u * step, capacity) : kNoSlot;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (s[u] == kNoSlot) continue;
            if (!RAISE) claim[s[u]] = (int)(i0 + u * step);
            else c[u] = *(volatile int*)(claim + s[u]);
        }
        if (RAISE) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (s[u] != kNoSlot && c[u] < (int)(i0 + u * step)) atomicMax(claim + s[u], (int)(i0 + u * step));
        }
    }
}

template <bool RAISE>
__global__ void sq_claim_kernel(const long long* slots, uint32_t n, uint32_t capacity, int* claim) {
    sq_claim_pass<RAISE>(slots, n, capacity, claim);
}

__global__ void __cluster_dims__(kClaimCtas, 1, 1) __launch_bounds__(kClaimThreads)
    sq_claim_cluster_kernel(const long long* slots, uint32_t n, uint32_t capacity, int* claim) {
    sq_claim_pass<false>(slots, n, capacity, claim);
    __threadfence();
    __syncthreads();
    asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
    sq_claim_pass<true>(slots, n, capacity, claim);
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

template <typename T, int BITS, int MODE, int TEAM, int CH>
cudaError_t go_write(const SqWrite& p, cudaStream_t st) {
    const int64_t per = kSqThreads / TEAM, items = (int64_t)p.n * p.groups;
    const int grid = (int)std::min<int64_t>((items + per - 1) / per, (int64_t)sm_count() * 32);
    note_launch();
    sq_write_kernel<T, BITS, MODE, TEAM, CH><<<grid, kSqThreads, 0, st>>>(p);
    return cudaGetLastError();
}

// The fewest lanes a group that leave each lane at most 4 chunks (8 for the
// longest groups), so that few shuffles join the maxima and a lane has several
// loads in flight; longer groups take a block.
template <typename T, int BITS, int MODE>
cudaError_t launch_write(const SqWrite& p, cudaStream_t st) {
    constexpr int E = sq_chunk<T, BITS, MODE>();
    const int chunks = (std::min(p.group, p.d) + E - 1) / E;
    if constexpr (MODE == kSqSingle) {
        if (chunks <= 16) return go_write<T, BITS, MODE, 4, 4>(p, st);
        if (chunks <= 64) return go_write<T, BITS, MODE, 16, 4>(p, st);
        if (chunks <= 256) return go_write<T, BITS, MODE, 32, 8>(p, st);
    } else {
        if (chunks <= 1) return go_write<T, BITS, MODE, 1, 1>(p, st);
        if (chunks <= 2) return go_write<T, BITS, MODE, 2, 1>(p, st);
        if (chunks <= 4) return go_write<T, BITS, MODE, 4, 1>(p, st);
        if (chunks <= 8) return go_write<T, BITS, MODE, 4, 2>(p, st);
        if (chunks <= 12) return go_write<T, BITS, MODE, 4, 3>(p, st);
        if (chunks <= 16) return go_write<T, BITS, MODE, 4, 4>(p, st);
        if (chunks <= 24) return go_write<T, BITS, MODE, 8, 3>(p, st);
        if (chunks <= 32) return go_write<T, BITS, MODE, 8, 4>(p, st);
        if (chunks <= 64) return go_write<T, BITS, MODE, 16, 4>(p, st);
        if (chunks <= 128) return go_write<T, BITS, MODE, 32, 4>(p, st);
        if (chunks <= 256) return go_write<T, BITS, MODE, 32, 8>(p, st);
    }
    const int grid = (int)std::min<int64_t>((int64_t)p.n * p.groups, (int64_t)sm_count() * 8);
    note_launch();
    if (chunks <= 2 * kSqThreads) sq_write_long_kernel<T, BITS, MODE, 2><<<grid, kSqThreads, 0, st>>>(p);
    else if (MODE == kSqShifted && chunks <= 4 * kSqThreads)
        sq_write_long_kernel<T, BITS, MODE, MODE == kSqShifted ? 4 : 8><<<grid, kSqThreads, 0, st>>>(p);
    else sq_write_long_kernel<T, BITS, MODE, 8><<<grid, kSqThreads, 0, st>>>(p);
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
        if (p.n <= kClaimRows) {
            note_launch();
            sq_claim_cluster_kernel<<<kClaimCtas, kClaimThreads, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
        } else {
            const int grid = (int)std::min<int64_t>(((int64_t)p.n + 255) / 256, (int64_t)sm_count() * 16);
            note_launch(2);
            sq_claim_kernel<false><<<grid, 256, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
            sq_claim_kernel<true><<<grid, 256, 0, st>>>(p.slots, p.n, p.capacity, p.claim);
        }
        const cudaError_t e = cudaGetLastError();
        if (e) return e;
    }
    const int es = type == kSqF32 ? 4 : 2;
    // a 16-byte chunk of values makes 4 or 8 (8 bits), 2 or 4 (4 bits) bytes of
    // codes.  Rows of x that are not aligned (an odd d, a slice) are put together from
    // aligned pieces: 45283 x 574 fp16 written and read back takes 70 us (the write 45 us), 166 us
    // value by value; the floor is 24 us.  Every piece is loaded by two neighbouring lanes
    const size_t cw = (size_t)(16 / es) * bits / 8;
    const bool codes = aligned(p.codes, cw) && p.ldc % cw == 0;
    const bool vec = codes && aligned(p.x, 16) && ((int64_t)p.ldx * es) % 16 == 0 && (p.d * es) % 16 == 0;
    auto go = [&](auto t, auto b) {
        using T = decltype(t);
        constexpr int BITS = decltype(b)::value;
        if (vec) return launch_write<T, BITS, kSqVec>(p, st);
        if (codes) return launch_write<T, BITS, kSqShifted>(p, st);
        return launch_write<T, BITS, kSqSingle>(p, st);
    };
    return by_type(type, [&](auto t) {
        return bits == 8 ? go(t, std::integral_constant<int, 8>{}) : go(t, std::integral_constant<int, 4>{});
    });
}

}  // namespace isb
