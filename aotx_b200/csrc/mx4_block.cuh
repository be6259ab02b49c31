// A block of 32 values in MX4: its scale and its codes.
#pragma once

#include "mx4_ptx.cuh"
#include "q8_common.cuh"

namespace q8 {

// The scale's byte for a block whose largest magnitude has these bits (of a float without its sign; a NaN is above
// everything): 2^(floor(log2 a) - 2), no smaller than 2^-127; 255 where the block is not finite.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t largest)
{
    const uint32_t exponent = largest >> 23;
    return exponent == 255u ? 255u : (exponent > 2u ? exponent - 2u : 0u);
}

// One over the scale: a power of two from 2^127 to 2^-125.
__device__ __forceinline__ float mx4_inverse(uint32_t scale)
{
    return __uint_as_float((254u - (scale != 255u ? scale : 0u)) << 23);
}

// The scale itself: 2^(scale - 127), of which the smallest is half of the smallest normal float; 255 is NaN.
__device__ __forceinline__ float mx4_scale_value(uint32_t scale)
{
    return __uint_as_float(scale == 255u ? 0x7FC00000u : (scale == 0u ? 0x00400000u : scale << 23));
}

// Eight values in a row: from memory (`aligned`: they lie on a 16-byte boundary), the largest magnitude of two such eights as
// mx4_scale takes it, their codes.
template <typename T>
struct Eight;

template <>
struct Eight<float> {
    uint4 a, b;
    __device__ __forceinline__ void zero()
    {
        a = b = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void load(const float *p, bool aligned)
    {
        if (aligned) {
            a = *reinterpret_cast<const uint4 *>(p);
            b = *reinterpret_cast<const uint4 *>(p + 4);
        } else {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(p);
            a = make_uint4(w[0], w[1], w[2], w[3]);
            b = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    // (as whole numbers, in which a NaN is above everything)
    __device__ __forceinline__ uint32_t largest() const
    {
        const uint32_t m = 0x7FFFFFFFu;
        return max(max(max(a.x & m, a.y & m), max(a.z & m, a.w & m)), max(max(b.x & m, b.y & m), max(b.z & m, b.w & m)));
    }
    static __device__ __forceinline__ uint32_t largest(const Eight &one, const Eight &two)
    {
        return max(one.largest(), two.largest());
    }
    __device__ __forceinline__ uint32_t codes(uint32_t scale, float inverse) const
    {
        const float v[8] = {__uint_as_float(a.x) * inverse, __uint_as_float(a.y) * inverse, __uint_as_float(a.z) * inverse,
                            __uint_as_float(a.w) * inverse, __uint_as_float(b.x) * inverse, __uint_as_float(b.y) * inverse,
                            __uint_as_float(b.z) * inverse, __uint_as_float(b.w) * inverse};
        return scale != 255u ? cvt_e2m1x8(v) : 0u;
    }
};

struct Eight16 {
    uint32_t w[4];
    __device__ __forceinline__ void zero()
    {
        w[0] = w[1] = w[2] = w[3] = 0u;
    }
    __device__ __forceinline__ void load(const void *p, bool aligned)
    {
        if (aligned) {
            const uint4 a = *static_cast<const uint4 *>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
            const unsigned short *h = static_cast<const unsigned short *>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = (uint32_t)h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
            }
        }
    }
    // The largest 15-bit magnitude, two halves of a word at a time (of binary16 and of bfloat16 alike, whole numbers order them).
    __device__ __forceinline__ uint32_t largest() const
    {
        const uint32_t m = 0x7FFF7FFFu;
        return __vmaxu2(__vmaxu2(w[0] & m, w[1] & m), __vmaxu2(w[2] & m, w[3] & m));
    }
    static __device__ __forceinline__ uint32_t magnitude(const Eight16 &one, const Eight16 &two)
    {
        const uint32_t both = __vmaxu2(one.largest(), two.largest());
        return max(both & 0xFFFFu, both >> 16);
    }
};

template <>
struct Eight<__half> : Eight16 {
    static __device__ __forceinline__ uint32_t largest(const Eight &one, const Eight &two)
    {
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)magnitude(one, two))));
    }
    __device__ __forceinline__ uint32_t codes(uint32_t scale, float inverse) const
    {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x * inverse, v[2 * i + 1] = f.y * inverse;
        }
        return scale != 255u ? cvt_e2m1x8(v) : 0u;
    }
};

template <>
struct Eight<__nv_bfloat16> : Eight16 {
    static __device__ __forceinline__ uint32_t largest(const Eight &one, const Eight &two)
    {
        return magnitude(one, two) << 16;
    }
    __device__ __forceinline__ uint32_t codes(uint32_t scale, float inverse) const
    {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16) * inverse, v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u) * inverse;
        }
        return scale != 255u ? cvt_e2m1x8(v) : 0u;
    }
};

} // namespace q8
