// sq.cuh -- device building blocks of the scalar-quantised rows, shared by sq.cu
// (write, read) and sq_mm.cu (the product that quantises its own tokens).
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

// values per chunk: 16 bytes of the floating type, or the fewest that fill a byte of codes
template <typename T, int BITS, bool VEC>
__host__ __device__ constexpr int sq_chunk() {
    return VEC ? 16 / (int)sizeof(T) : 8 / BITS;
}

// item = row * parts + part
__device__ __forceinline__ void sq_split(int64_t item, int parts, int64_t& row, int& part) {
    if (parts == 1) {
        row = item;
        part = 0;
    } else if (item < (int64_t(1) << 32)) {
        const uint32_t r = (uint32_t)item / (uint32_t)parts;
        row = r;
        part = (int)((uint32_t)item - r * (uint32_t)parts);
    } else {
        row = item / parts;
        part = (int)(item - row * parts);
    }
}

// values e0 .. e0 + E - 1 of a group of `width` values, 0 past its end
template <typename T, bool VEC, int E>
__device__ __forceinline__ void sq_load(const T* __restrict__ x, int e0, int width, float (&v)[E]) {
    if (VEC && e0 + E <= width) {
        const uint4 raw = *reinterpret_cast<const uint4*>(x + e0);
        T t[16 / sizeof(T)];
        memcpy(t, &raw, 16);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = sq_float(t[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e0 + e < width ? sq_float(x[e0 + e]) : 0.f;
    }
}

struct SqScale {
    float scale;   // as stored
    float inv;     // 1 / scale rounded; 0 where every code is 0 (scale 0, infinite or NaN)
    float half;    // scale / 2
};

// the scale of a group from the bits of its largest |x|.  The maximum is taken
// over bit patterns: there NaN > infinity > every number.
template <int BITS>
__device__ __forceinline__ SqScale sq_scale(uint32_t top) {
    SqScale s;
    s.scale = __fdiv_rn(__uint_as_float(top), BITS == 8 ? 127.f : 7.f);
    const bool none = !(s.scale > 0.f && s.scale < __int_as_float(0x7f800000));
    s.inv = none ? 0.f : __frcp_rn(s.scale);
    s.half = 0.5f * s.scale;
    return s;
}

// Codes of E values: round-half-even(x / scale), exactly as the quotient of real
// numbers rounds.  x * inv is within 2^-22 of the quotient, so its rounding k is
// off by one at most, and only next to a border between two codes.  The
// remainder r = x - k scale is a multiple of the smaller of the two numbers'
// last places and at most about scale / 2, so the fused multiply-add gives it
// exactly: |r| < scale / 2 proves k, anything else (rare) is put right there.
// 1.5 * 2^23 is added so that the sum's last bits are k itself.
// Scales below 2^-100 (where half a step or 1 / scale leaves fp32's range) divide in fp64,
// whose quotient of two fp32 numbers cannot round onto a border it is not on:
// the two are 2^-33 apart at least, relative to the quotient.
template <int BITS, int E>
__device__ __forceinline__ void sq_codes(const float (&v)[E], const SqScale& s, uint32_t (&k)[E]) {
    constexpr float kMagic = 12582912.f;
    if (s.inv == 0.f) {
#pragma unroll
        for (int e = 0; e < E; ++e) k[e] = 0;
        return;
    }
    if (s.scale < 7.888609e-31f) {
        const double L = BITS == 8 ? 127.0 : 7.0;
#pragma unroll
        for (int e = 0; e < E; ++e)
            k[e] = (uint32_t)(int)fmin(fmax(rint((double)v[e] / (double)s.scale), -L), L);
        return;
    }
    float far = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float t = __fmaf_rn(v[e], s.inv, kMagic);
        k[e] = __float_as_uint(t);
        far = fmaxf(far, fabsf(__fmaf_rn(-(t - kMagic), s.scale, v[e])));
    }
    if (far >= s.half) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float t = __uint_as_float(k[e]) - kMagic;
            const float r = __fmaf_rn(-t, s.scale, v[e]);
            const int i = (int)t;
            k[e] = (uint32_t)(r > s.half || (r == s.half && (i & 1))      ? i + 1
                              : r < -s.half || (r == -s.half && (i & 1)) ? i - 1
                                                                         : i);
        }
    }
}

// stores the codes of values e0 .. e0 + E - 1 of a group of `width` values at
// cr (the group's first byte)
template <int BITS, bool VEC, int E>
__device__ __forceinline__ void sq_store(uint8_t* cr, int e0, int width, const float (&v)[E], const SqScale& s) {
    uint32_t k[E];
    sq_codes<BITS, E>(v, s, k);
    constexpr int W = E * BITS / 8;              // bytes of a chunk
    uint8_t by[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        by[w] = BITS == 8 ? (uint8_t)k[w] : (uint8_t)((k[2 * w % E] & 15u) | ((k[(2 * w + 1) % E] & 15u) << 4));
    const int b0 = e0 * BITS / 8;
    if (VEC && e0 + E <= width) {
        if constexpr (W == 8) *reinterpret_cast<uint2*>(cr + b0) = *reinterpret_cast<uint2*>(by);
        else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(cr + b0) = *reinterpret_cast<uint32_t*>(by);
        else if constexpr (W == 2) *reinterpret_cast<uint16_t*>(cr + b0) = *reinterpret_cast<uint16_t*>(by);
        else cr[b0] = by[0];
    } else {
        // values past the group's end are 0, so the last odd value's byte has an empty high half
#pragma unroll
        for (int w = 0; w < W; ++w)
            if (e0 + w * 8 / BITS < width) cr[b0 + w] = by[w];
    }
}

// W bytes of codes from byte b0 of a row of `bytes` bytes, 0 past its end
template <bool VEC, int W>
__device__ __forceinline__ void sq_load_codes(const uint8_t* __restrict__ cr, int b0, int bytes, uint8_t (&q)[W]) {
    if (VEC && b0 + W <= bytes) {
        if constexpr (W == 8) *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(cr + b0);
        else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(q) = *reinterpret_cast<const uint32_t*>(cr + b0);
        else if constexpr (W == 2) *reinterpret_cast<uint16_t*>(q) = *reinterpret_cast<const uint16_t*>(cr + b0);
        else q[0] = cr[b0];
    } else {
#pragma unroll
        for (int w = 0; w < W; ++w) q[w] = b0 + w < bytes ? cr[b0 + w] : (uint8_t)0;
    }
}

template <int BITS>
__device__ __forceinline__ int sq_code(const uint8_t* q, int e) {
    if (BITS == 8) return (int)(int8_t)q[e];
    return (int)((int8_t)(uint8_t)(q[e >> 1] << (e & 1 ? 0 : 4)) >> 4);
}

template <typename T, bool VEC, int E>
__device__ __forceinline__ void sq_store_values(T* out, int e0, int d, const float (&v)[E]) {
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sq_round(v[e], t[e]);
    if (VEC && e0 + E <= d) {
        uint4 raw;
        memcpy(&raw, t, 16);
        *reinterpret_cast<uint4*>(out + e0) = raw;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e0 + e < d) out[e0 + e] = t[e];
    }
}

}  // namespace isb
