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

__device__ __forceinline__ uint32_t mx4_codes(float (&v)[8], uint32_t scale, float inverse)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] *= inverse;
    }
    return scale != 255u ? cvt_e2m1x8(v) : 0u;
}

__device__ __forceinline__ uint32_t mx4_largest(const float (&v)[8], uint32_t largest)
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        largest = max(largest, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    }
    return largest;
}

// Eight values in a row, from memory and as floats; `aligned`: they lie on a 16-byte boundary.
template <typename T>
struct Eight;

template <>
struct Eight<float> {
    uint4 a, b;
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
    __device__ __forceinline__ void floats(float (&v)[8]) const
    {
        v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z), v[3] = __uint_as_float(a.w);
        v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y), v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
    }
};

struct Eight16 {
    uint32_t w[4];
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
};

template <>
struct Eight<__half> : Eight16 {
    __device__ __forceinline__ void floats(float (&v)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
};

template <>
struct Eight<__nv_bfloat16> : Eight16 {
    __device__ __forceinline__ void floats(float (&v)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};

} // namespace q8
