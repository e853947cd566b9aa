// Eight halves divided by a scale and rounded to int8: the cache's elements, and the queries that choose among its blocks.
#pragma once

#include "common.cuh"

namespace pplb200 {
namespace {

union Eight {
    uint4 raw;
    __half2 h[4];
};

// Quotients by one scale, rounded to nearest even, as bytes.  Their magnitude is at most 127.07 (65504 / 515.5, the cache's largest scale).  The product with the scale's
// reciprocal, moved by 2^-21 to either side, brackets the quotient in 32 bits (the reciprocal is off by 2^-23 at most, its moving, the
// product and the quotient by 2^-24 each); 1.5 * 2^23 added, the low byte is the rounded number.  Where the two sides differ, and in a
// group with an infinity or a NaN, the division decides; there NaN becomes 0, and is NaN again when it is multiplied by that group's scale.
struct Quotient {
    float s, hi, lo;
    uint32_t special;
    __device__ __forceinline__ explicit Quotient(half scale) {
        s = __half2float(scale);
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
        hi = inv * (1.0f + 0x1p-21f);
        lo = inv * (1.0f - 0x1p-21f);
        special = __half_as_ushort(scale) < 0x7c00u ? 0u : 1u;
    }
    __device__ __forceinline__ uint2 eight(const Eight& e) const {
        constexpr float kMagic = 12582912.0f;
        uint32_t b[8], differ = special;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(e.h[i]);
            b[2 * i] = __float_as_uint(__fmaf_rn(v.x, hi, kMagic));
            b[2 * i + 1] = __float_as_uint(__fmaf_rn(v.y, hi, kMagic));
            differ |= b[2 * i] ^ __float_as_uint(__fmaf_rn(v.x, lo, kMagic));
            differ |= b[2 * i + 1] ^ __float_as_uint(__fmaf_rn(v.y, lo, kMagic));
        }
        if (differ != 0u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = __half22float2(e.h[i]);
                b[2 * i] = (uint32_t)__float2int_rn(__fdiv_rn(v.x, s));
                b[2 * i + 1] = (uint32_t)__float2int_rn(__fdiv_rn(v.y, s));
            }
        }
        return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                          __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
    }
};

} // namespace
} // namespace pplb200
