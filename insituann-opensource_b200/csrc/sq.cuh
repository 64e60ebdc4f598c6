// sq.cuh -- device building blocks of the scalar-quantised rows, shared by
// sq_write.cu, sq_read.cu and sq_mm.cu (whose product quantises few tokens itself).
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
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

namespace isb {

__device__ __forceinline__ float sq_float(float x) { return x; }
__device__ __forceinline__ float sq_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float sq_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void sq_round(float v, float& o) { o = v; }
__device__ __forceinline__ void sq_round(float v, __half& o) { o = __float2half_rn(v); }
__device__ __forceinline__ void sq_round(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// How floating rows are taken, a chunk at a time:
//   kSqVec      rows are 16-byte aligned and a whole number of chunks of 16 bytes
//               long: a chunk is inside its group or outside
//   kSqShifted  rows of any alignment, in chunks of 16 bytes put together from
//               aligned pieces; a group's last chunk may be a part (the codes
//               are aligned as for kSqVec)
//   kSqSingle   chunks of the fewest values that fill a byte of codes
constexpr int kSqSingle = 0, kSqVec = 1, kSqShifted = 2;

template <typename T, int BITS, int MODE>
__host__ __device__ constexpr int sq_chunk() {
    return MODE != kSqSingle ? 16 / (int)sizeof(T) : 8 / BITS;
}

constexpr uint32_t kNoSlot = 0xffffffffu;

// slot of a row, kNoSlot outside the store
__device__ __forceinline__ uint32_t sq_slot(const long long* __restrict__ slots, uint32_t row, uint32_t capacity) {
    if (!slots) return row;
    const unsigned long long s = (unsigned long long)slots[row];
    return s < capacity ? (uint32_t)s : kNoSlot;
}

// item = row * parts + part
__device__ __forceinline__ void sq_split(uint64_t item, int parts, uint32_t& row, int& part) {
    if (parts == 1) {
        row = (uint32_t)item;
        part = 0;
    } else if (item >> 32 == 0) {
        row = (uint32_t)item / (uint32_t)parts;
        part = (int)((uint32_t)item - row * (uint32_t)parts);
    } else {
        row = (uint32_t)(item / (uint32_t)parts);
        part = (int)(item - (uint64_t)row * (uint32_t)parts);
    }
}

// two fp32 operations in one instruction, each rounded as its scalar form
__device__ __forceinline__ float2 sq_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
        " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 sq_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
        " add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 sq_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n"
        " mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 16 bytes of a row in flight: issue() starts the loads and has no branch, so
// that several of them are under way at once; take() gives the bytes.  ALIGNED:
// rows are 16-byte aligned, and what follows a row's end is what lies there;
// else the two aligned 16-byte pieces around the bytes are read and shifted, and
// 0 follows a row's end.  A piece that is not wholly inside the array [lo, hi)
// (at its ends only) is read by bytes.
template <bool ALIGNED>
struct SqBytes {
    uint32_t v[ALIGNED ? 4 : 8];

    // bytes [at, at + 16) of a row that ends at `end` (at >= end: none)
    __device__ __forceinline__ void issue(uintptr_t at, uintptr_t end, uintptr_t lo, uintptr_t hi) {
        if constexpr (ALIGNED) {
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (at < end && at + 16 <= hi) x = __ldg(reinterpret_cast<const uint4*>(at));
            v[0] = x.x;
            v[1] = x.y;
            v[2] = x.z;
            v[3] = x.w;
        } else {
            const uintptr_t w = at & ~uintptr_t(15);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 x = make_uint4(0u, 0u, 0u, 0u);
                if (at < end && w + 16 * h < end && w + 16 * h >= lo && w + 16 * h + 16 <= hi)
                    x = __ldg(reinterpret_cast<const uint4*>(w + 16 * h));
                v[4 * h] = x.x;
                v[4 * h + 1] = x.y;
                v[4 * h + 2] = x.z;
                v[4 * h + 3] = x.w;
            }
        }
    }
    __device__ __forceinline__ uint4 take(uintptr_t at, uintptr_t end, uintptr_t lo, uintptr_t hi) {
        if constexpr (ALIGNED) {
            if (at < end && at + 16 > hi) {                      // the last bytes of the array
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = edge(at + 4 * i, lo, hi);
            }
            return make_uint4(v[0], v[1], v[2], v[3]);
        } else {
            const uintptr_t w = at & ~uintptr_t(15);
            if (at < end && (w < lo || w + 32 > hi)) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (w + (i & 4) * 4 < lo || w + (i & 4) * 4 + 16 > hi) v[i] = edge(w + 4 * i, lo, hi);
            }
            const uint4 x = shifted(at);
            uint32_t o[4] = {x.x, x.y, x.z, x.w};
            if (at + 16 > end) clear(o, at < end ? (int)(end - at) : 0);
            return make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    // the same for a row with 16 bytes of the array before and behind it, `left` bytes from at to its end (at most
    // 0: none): no piece leaves the array, and the tests are of 32 bits
    __device__ __forceinline__ void issue_inner(uintptr_t at, int left) {
        const uint4* w = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
        uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
        if (left > 0) x = __ldg(w);
        if (left > 16 - (int)(at & 15)) y = __ldg(w + 1);
        v[0] = x.x;
        v[1] = x.y;
        v[2] = x.z;
        v[3] = x.w;
        v[4] = y.x;
        v[5] = y.y;
        v[6] = y.z;
        v[7] = y.w;
    }
    __device__ __forceinline__ uint4 take_inner(uintptr_t at, int left) {
        const uint4 x = shifted(at);
        if (left >= 16) return x;
        uint32_t o[4] = {x.x, x.y, x.z, x.w};
        clear(o, left);
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
    // clears the bytes from `left` on
    static __device__ __forceinline__ void clear(uint32_t (&o)[4], int left) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = left - 4 * i;
            o[i] = n >= 4 ? o[i] : n <= 0 ? 0u : o[i] & ((1u << (8 * n)) - 1u);
        }
    }
    // the 16 bytes from at & 15 on: by two words, by one, by bits
    __device__ __forceinline__ uint4 shifted(uintptr_t at) {
        const bool two = (at & 8) != 0, one = (at & 4) != 0;
#pragma unroll
        for (int i = 0; i < 6; ++i) v[i] = two ? v[i + 2] : v[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) v[i] = one ? v[i + 1] : v[i];
        const uint32_t sh = (uint32_t)(at & 3) * 8;
        return make_uint4(__funnelshift_r(v[0], v[1], sh), __funnelshift_r(v[1], v[2], sh),
                          __funnelshift_r(v[2], v[3], sh), __funnelshift_r(v[3], v[4], sh));
    }
    // the word at w, 0 where its bytes are outside [lo, hi)
    static __device__ __forceinline__ uint32_t edge(uintptr_t w, uintptr_t lo, uintptr_t hi) {
        uint32_t x = 0;
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
            if (w + i >= lo && w + i < hi) x |= (uint32_t)*reinterpret_cast<const uint8_t*>(w + i) << (8 * i);
        return x;
    }
};

// ---- floating chunks, kept as they were read (half the registers of fp32 for
// the 16-bit types) ----
template <typename T, int E>
struct SqRaw {
    static constexpr int kWords = (E * (int)sizeof(T) + 3) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else {
            const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            T t;
            memcpy(&t, &h, 2);
            return sq_float(t);
        }
    }
    // raises `top` (bit patterns of |x|, two 16-bit halves apart or one 32-bit) by this chunk's
    __device__ __forceinline__ void top(uint32_t& t) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            t = sizeof(T) == 4 ? max(t, w[i] & 0x7fffffffu) : __vmaxu2(t, w[i] & 0x7fff7fffu);
    }
};

// 16 bytes at the ends of the array, out of line: the first and the last row
// take this way only, and a small call's time is reading its instructions
static __device__ __noinline__ uint4 sq_end_bytes(uintptr_t at, uintptr_t end, uintptr_t lo, uintptr_t hi) {
    SqBytes<false> b;
    b.issue(at, end, lo, hi);
    return b.take(at, end, lo, hi);
}

// the bytes of all rows, and whether 16 of them lie before and behind the group at hand
struct SqSpan {
    uintptr_t lo, hi;
    bool inner;
    template <typename T>
    __device__ __forceinline__ void at(const T* x, int width) {
        inner = reinterpret_cast<uintptr_t>(x) - lo >= 16 && hi - reinterpret_cast<uintptr_t>(x + width) >= 16;
    }
};

// Values e0 .. e0 + E - 1 of a group of `width` values at x, 0 past its end:
// issue() starts the loads, take() gives the values.
template <typename T, int MODE, int E>
struct SqLoad {
    SqRaw<T, E> r;
    __device__ __forceinline__ void issue(const T* __restrict__ x, int e0, int width, const SqSpan&) {
#pragma unroll
        for (int i = 0; i < SqRaw<T, E>::kWords; ++i) r.w[i] = 0;
        if constexpr (MODE == kSqVec) {
            if (e0 < width) {
                const uint4 v = *reinterpret_cast<const uint4*>(x + e0);
                memcpy(r.w, &v, sizeof(r.w));
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e0 + e < width) {
                    if constexpr (sizeof(T) == 4) r.w[e] = reinterpret_cast<const uint32_t*>(x)[e0 + e];
                    else r.w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(x)[e0 + e] << (16 * (e & 1));
                }
        }
    }
    __device__ __forceinline__ SqRaw<T, E> take(const T*, int, int, const SqSpan&) { return r; }
};

template <typename T, int E>
struct SqLoad<T, kSqShifted, E> {
    SqBytes<false> b;
    __device__ __forceinline__ void issue(const T* x, int e0, int width, const SqSpan& s) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(x + e0);
        b.issue_inner(at, s.inner ? (width - e0) * (int)sizeof(T) : 0);
    }
    __device__ __forceinline__ SqRaw<T, E> take(const T* x, int e0, int width, const SqSpan& s) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(x + e0);
        uint4 v = b.take_inner(at, (width - e0) * (int)sizeof(T));
        if (!s.inner && e0 < width) v = sq_end_bytes(at, reinterpret_cast<uintptr_t>(x + width), s.lo, s.hi);
        SqRaw<T, E> r;
        memcpy(r.w, &v, sizeof(r.w));
        return r;
    }
};

// |x| as fp32 bits from the bit pattern that SqRaw::top raised (halves joined).
// The maximum is taken over bit patterns: there NaN > infinity > every number.
template <typename T>
__device__ __forceinline__ float sq_top(uint32_t t) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(t);
    else {
        const uint16_t h = (uint16_t)max(t >> 16, t & 0xffffu);
        T v;
        memcpy(&v, &h, 2);
        return sq_float(v);
    }
}

struct SqScale {
    float scale;   // as stored
    float inv;     // 1 / scale rounded; 0 where every code is 0 (scale 0, infinite or NaN)
    float half;    // a remainder of at least this asks for the slow quotient
};

// Scales below 2^-100 (where half a step or 1 / scale leaves fp32's range) always take the slow quotient.
template <int BITS>
__device__ __forceinline__ SqScale sq_scale(float top) {
    SqScale s;
    s.scale = __fdiv_rn(top, BITS == 8 ? 127.f : 7.f);
    const float inf = __int_as_float(0x7f800000);
    const bool none = !(s.scale > 0.f && s.scale < inf);
    s.inv = none ? 0.f : __frcp_rn(s.scale);
    s.half = none ? inf : s.scale < 7.888609e-31f ? 0.f : 0.5f * s.scale;
    return s;
}

// round-half-even(x / scale) in fp64, whose quotient of two fp32 numbers cannot
// round onto a border between codes that it is not on: the two are 2^-33 apart at
// least, relative to the quotient.
template <int BITS>
__device__ __noinline__ uint32_t sq_code_slow(float x, float scale) {
    const double L = BITS == 8 ? 127.0 : 7.0;
    return (uint32_t)(int)fmin(fmax(rint((double)x / (double)scale), -L), L);
}

// Codes of E values, packed as the store holds them: round-half-even(x / scale),
// exactly as the quotient of real numbers rounds.  x * inv is within 2^-22 of
// the quotient (relative), so its rounding k is off by one at most, and only next
// to a border between two codes.  The remainder r = x - k scale is a multiple
// of the smaller of the two numbers' last places and at most about scale / 2,
// so the fused multiply-add gives it exactly: |r| < scale / 2 proves k; beyond it k
// is one off, and on it the even neighbour is the code (both rare: one in
// some 10^5 values).  1.5 * 2^23 is added so that the sum's last bits are k itself.
// Where 1 / scale is infinite a zero makes r NaN; fmaxf passes over it, and `far`
// of 0 reaches the half of 0 that such a scale has.
template <typename T, int BITS, int E>
__device__ __forceinline__ void sq_codes(const SqRaw<T, E>& x, const SqScale& s, uint32_t (&q)[(E * BITS + 31) / 32]) {
    constexpr float kMagic = 12582912.f;
    uint32_t k[E];
    float far = 0.f;
    if constexpr (E == 1) {
        const float v = x.get(0);
        const float t = __fmaf_rn(v, s.inv, kMagic);
        k[0] = __float_as_uint(t);
        far = fmaxf(far, fabsf(__fmaf_rn(kMagic - t, s.scale, v)));
    } else {
        const float2 inv = make_float2(s.inv, s.inv), sc = make_float2(-s.scale, -s.scale);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 v = make_float2(x.get(e), x.get(e + 1));
            const float2 t = sq_fma2(v, inv, make_float2(kMagic, kMagic));
            k[e] = __float_as_uint(t.x);
            k[e + 1] = __float_as_uint(t.y);
            const float2 r = sq_fma2(sq_add2(t, make_float2(-kMagic, -kMagic)), sc, v);
            far = fmaxf(far, fmaxf(fabsf(r.x), fabsf(r.y)));
        }
    }
    if (far >= s.half) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = x.get(e), t = __uint_as_float(k[e]) - kMagic, r = __fmaf_rn(-t, s.scale, v);
            const int i = (int)t, odd = i & 1;
            if (s.half == 0.f) k[e] = sq_code_slow<BITS>(v, s.scale);
            else k[e] = (uint32_t)(i + (r > s.half || (r == s.half && odd)) - (r < -s.half || (r == -s.half && odd)));
        }
    }
    if constexpr (BITS == 8 && E % 4 == 0) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i)
            q[i] = __byte_perm(__byte_perm(k[4 * i], k[4 * i + 1], 0x0040),
                               __byte_perm(k[4 * i + 2], k[4 * i + 3], 0x0040), 0x5410);
    } else {
        q[0] = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) q[0] |= (k[e] & ((1u << BITS) - 1u)) << (BITS * e);
    }
    // infinities and NaN reach the sums above: their groups' codes are 0 by choice
#pragma unroll
    for (int i = 0; i < (E * BITS + 31) / 32; ++i) q[i] = s.inv == 0.f ? 0u : q[i];
}

// stores the codes of values e0 .. e0 + E - 1 of a group of `width` values (e0 <
// width) at cr (the group's first byte); values past the group's end are 0, so
// the last odd value's byte has an empty high half
template <typename T, int BITS, int MODE, int E>
__device__ __forceinline__ void sq_store(uint8_t* cr, int e0, int width, const SqRaw<T, E>& x, const SqScale& s) {
    uint32_t q[(E * BITS + 31) / 32];
    sq_codes<T, BITS, E>(x, s, q);
    constexpr int W = E * BITS / 8;              // bytes of a chunk
    uint8_t* to = cr + e0 * BITS / 8;
    if constexpr (MODE == kSqShifted) {
        if (e0 + E > width) {
#pragma unroll
            for (int w = 0; w < W; ++w)
                if (e0 + w * 8 / BITS < width) to[w] = (uint8_t)(q[w >> 2] >> (8 * (w & 3)));
            return;
        }
    }
    if constexpr (W == 8) *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
    else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(to) = q[0];
    else if constexpr (W == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)q[0];
    else to[0] = (uint8_t)q[0];
}

// W bytes of codes
template <int W>
__device__ __forceinline__ void sq_load_codes(const uint8_t* __restrict__ cr, uint32_t (&q)[(W + 3) / 4]) {
    if constexpr (W == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(cr);
        q[0] = v.x;
        q[1] = v.y;
    } else if constexpr (W == 4) q[0] = *reinterpret_cast<const uint32_t*>(cr);
    else if constexpr (W == 2) q[0] = *reinterpret_cast<const uint16_t*>(cr);
    else q[0] = cr[0];
}

// the values of E codes.  A code c is put into the last bits of 2^23 (as c + 128,
// or c + 8), and 2^23 + 128 (+ 8) taken away: whole numbers, exact in fp32.
template <int BITS, int E>
__device__ __forceinline__ void sq_values(const uint32_t (&q)[(E * BITS + 31) / 32], float scale, float (&v)[E]) {
    constexpr uint32_t kBase = 0x4b000000u;
    constexpr float kZero = BITS == 8 ? 8388736.f : 8388616.f;
    const uint32_t lo = (q[0] & 0x0f0f0f0fu) ^ 0x08080808u, hi = ((q[0] >> 4) & 0x0f0f0f0fu) ^ 0x08080808u;
#pragma unroll
    for (int e = 0; e < E; ++e)
        v[e] = __uint_as_float(BITS == 8 ? __byte_perm(q[e >> 2] ^ 0x80808080u, kBase, 0x7440 | (e & 3))
                                         : __byte_perm(e & 1 ? hi : lo, kBase, 0x7440 | (e >> 1)));
    if constexpr (E == 1) v[0] = (v[0] - kZero) * scale;
    else {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 r = sq_mul2(sq_add2(make_float2(v[e], v[e + 1]), make_float2(-kZero, -kZero)),
                                     make_float2(scale, scale));
            v[e] = r.x;
            v[e + 1] = r.y;
        }
    }
}

// values e0 .. e0 + E - 1 of a row of d values; `once`: the caches need not keep them
template <typename T, bool VEC, int E>
__device__ __forceinline__ void sq_store_values(T* out, int e0, int d, const float (&v)[E], bool once) {
    if constexpr (VEC && sizeof(T) == 2) {
        uint32_t w[E / 2];
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            T t[2];
            sq_round(v[2 * i], t[0]);
            sq_round(v[2 * i + 1], t[1]);
            memcpy(&w[i], t, 4);
        }
        const uint4 o = make_uint4(w[0], w[1], w[2], w[3]);
        if (once) __stcs(reinterpret_cast<uint4*>(out + e0), o);
        else *reinterpret_cast<uint4*>(out + e0) = o;
    } else if constexpr (VEC) {
        const float4 o = make_float4(v[0], v[1], v[2], v[3]);
        if (once) __stcs(reinterpret_cast<float4*>(out + e0), o);
        else *reinterpret_cast<float4*>(out + e0) = o;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e0 + e < d) sq_round(v[e], out[e0 + e]);
    }
}

}  // namespace isb
