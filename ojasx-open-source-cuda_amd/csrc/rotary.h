// rotary.h -- the rotation of positions: a pair's angle, and one pair turned by it.  Shared by the
// rotation of queries and keys (rotary.hip) and the cache's rotated append (kv8_cache.hip), whose
// keys are the same to the bit.
//
// Pair i of a head at position p turns by p * rate[i] / 2^64 of a whole turn: the product modulo 2^64
// is exact for whole positions of any size, so far positions lose nothing (an fp32 angle at position
// 10^6 is off by 0.06) and no table of cosines is read.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ojx {

// What turns a head's first 2 * pairs elements.
struct Rotation {
    const uint64_t* rates;  // [pairs], turns per position in 2^-64
    const void* positions;  // int32 or int64
    int wide;               // the latter
    int pairs;
    int interleaved;        // pairs (2i, 2i + 1), else (i, i + pairs)
    float cos_gain;         // factors of both: the gain, for the sine with the direction's sign
    float sin_gain;
};

__device__ __forceinline__ uint64_t position_at(const Rotation& r, int64_t i) {
    return r.wide ? (uint64_t) static_cast<const int64_t*>(r.positions)[i]
                  : (uint64_t)(int64_t) static_cast<const int32_t*>(r.positions)[i];
}

// Cosine and sine of phase / 2^64 turns.  The upper 32 bits (2^-29 of a radian) are a quadrant and a
// remainder within an eighth of a turn, whose Taylor polynomials (first terms left out: x^11 / 11! and
// x^12 / 12!, under 2^-29) are evaluated in fp32: off by 2^-22 at most, nearly all of it the rounding
// of the remainder.
__device__ __forceinline__ void turn_of(uint64_t phase, float& c, float& s) {
    const uint32_t f = (uint32_t)(phase >> 32);
    const uint32_t q = (f + 0x20000000u) >> 30;
    const float r = (float)(int32_t)(f - (q << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float z = r * r;
    float a = __builtin_fmaf(z, 2.75573192239858907e-6f, -1.98412698412698413e-4f);
    a = __builtin_fmaf(z, a, 8.33333333333333333e-3f);
    a = __builtin_fmaf(z, a, -1.66666666666666667e-1f);
    a = __builtin_fmaf(r * z, a, r);
    float b = __builtin_fmaf(z, -2.75573192239858907e-7f, 2.48015873015873016e-5f);
    b = __builtin_fmaf(z, b, -1.38888888888888889e-3f);
    b = __builtin_fmaf(z, b, 4.16666666666666667e-2f);
    b = __builtin_fmaf(z, b, -0.5f);
    b = __builtin_fmaf(z, b, 1.f);
    const bool odd = q & 1;
    c = __uint_as_float(__float_as_uint(odd ? a : b) ^ ((q + 1) & 2) << 30);
    s = __uint_as_float(__float_as_uint(odd ? b : a) ^ (q & 2) << 30);
}

// The pair's cosine and sine times their gains.
__device__ __forceinline__ void pair_turn(const Rotation& r, uint64_t position, uint64_t rate, float& c,
                                          float& s) {
    turn_of(position * rate, c, s);
    c *= r.cos_gain;
    s *= r.sin_gain;
}

__device__ __forceinline__ void turn_pair(float c, float s, float& lo, float& hi) {
    const float x = lo, y = hi;
    lo = __builtin_fmaf(x, c, -(y * s));
    hi = __builtin_fmaf(y, c, x * s);
}

}  // namespace ojx
