// Rows of 16- or 32-bit values to MX4 (E2M1 codes, a power of two per 32 values) and back.
//
//   a = max |x_i| over the block,  s = 2^max(floor(log2 a) - 2, -127),  c_i = E2M1(x_i / s), nearest, ties to even
//
// All of it is exact but the last rounding: s is read off the exponent of a, and the division by a power of two is a
// multiplication by another.  Two bytes a value in and half a byte out: memory bounds it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "mx4.h"
#include "mx4_block.cuh"
#include "q8_launch.h"

namespace q8 {

// A lane takes half a block, 16 values, so eight lanes a chunk of 128 with its word of four scales, and a warp the same chunk of
// four successive rows; a block 32 rows by kQuantChunks chunks, whose loads are issued together.  The largest magnitude of
// 16-bit values is found two at a time, and the products by the scale's reciprocal are formed two at a time too.  Instructions were
// what bound the first form of these kernels (eight values a lane, one at a time, 13 instructions a value; 28672 x 4096
// in binary16 there and back 112 us, now 98.5; quantisation alone 47.9, 6.2 TB/s).
constexpr uint32_t kQuantThreads = 256;
constexpr uint32_t kQuantRows = kQuantThreads / 8u;
constexpr uint32_t kQuantChunks = 4;

// OWN_PRODUCT: the launch behind is the product that the quantisation is part of, which may start at once (it reads x in MX4 behind its
// wait).  Else what is written may be weights, which a product reads without a wait: the kernel does not let its dependents go
// (griddepcontrol.launch_dependents is not in it), so nothing behind it starts before it has ended, and dependents need no wait
// for what it wrote.  (With dependents let go at the stores the product of 28672 x 4096 behind 300 rows is done 0.9 us sooner, of 37.9, and
// behind 1 or 8 rows no sooner; a routed layer's gate and up step of 512 tokens, let go behind the wait, 1 us, of 53.)
template <typename T, bool OWN_PRODUCT>
__global__ void __launch_bounds__(kQuantThreads)
mx4_quantize_kernel(const T *x, uint32_t x_rows, unsigned long long ldx, uint32_t k, const uint32_t *rows_of, uint32_t rows,
                    const uint32_t *rows_dev, uint2 *__restrict__ codes, uint8_t *__restrict__ scales, bool aligned)
{
    constexpr uint32_t kTogether = sizeof(T) == 4u ? 2u : kQuantChunks;
    if (OWN_PRODUCT) {
        grid_launch_dependents();
    }
    grid_dependency_wait();
    uint32_t live = rows;
    if (rows_dev != nullptr) {
        const uint32_t on_device = *rows_dev;
        live = on_device < rows ? on_device : rows;
    }
    const uint32_t row = blockIdx.x * kQuantRows + threadIdx.x / 8u;
    const uint32_t lane = threadIdx.x % 8u;
    uint32_t from = row;
    if (row < live && rows_of != nullptr) {
        from = rows_of[row];
    }
    // (all lanes go on: the exchanges below are among whole warps)
    const bool here = row < live && from < x_rows;
    const uint32_t chunks = here ? mx4_chunks(k) : 0u;
    const uint32_t first = blockIdx.y * kQuantChunks;
    const T *x_at = x + (here ? (unsigned long long)from * ldx : 0ull) + first * 128u + lane * 16u;
    uint2 *code_at = codes + (unsigned long long)row * (k / 16u) + first * 8u + lane;
    uint8_t *scale_at = scales + ((unsigned long long)first * rows + row) * 4u + lane / 2u;
#pragma unroll
    for (uint32_t c0 = 0; c0 < kQuantChunks; c0 += kTogether) {
        Eight<T> raw[kTogether][2];
#pragma unroll
        for (uint32_t i = 0; i < kTogether; ++i) {
            raw[i][0].zero();
            raw[i][1].zero();
            if (here && (first + c0 + i) * 128u + lane * 16u < k) {
                raw[i][0].load(x_at + (c0 + i) * 128u, aligned);
                raw[i][1].load(x_at + (c0 + i) * 128u + 8u, aligned);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kTogether; ++i) {
            const uint32_t c = first + c0 + i;
            uint32_t largest = Eight<T>::largest(raw[i][0], raw[i][1]);
            largest = max(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 1u));
            const uint32_t scale = mx4_scale(largest);
            const float inverse = mx4_inverse(scale);
            const uint2 word = make_uint2(raw[i][0].codes(scale, inverse), raw[i][1].codes(scale, inverse));
            const bool in = c * 128u + lane * 16u < k;
            if (here && in) {
                code_at[(c0 + i) * 8u] = word;
            }
            if (c < chunks && (lane & 1u) == 0u) {
                scale_at[(unsigned long long)(c0 + i) * rows * 4u] = (uint8_t)(in ? scale : 0u);   // (0 past k)
            }
        }
    }
}

// Values (pairs of halves) by their scale, as 16 bytes of T.
__device__ __forceinline__ uint4 mx4_put(const uint32_t (&halves)[4], uint32_t scale, __half)
{
    uint32_t word[4];
    if (scale - 114u <= 25u) {
        // 2^-13 .. 2^12: the product of two halves is exact
        const __half2 by = __half2half2(__ushort_as_half((unsigned short)((scale - 112u) << 10)));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 v = __hmul2(*reinterpret_cast<const __half2 *>(&halves[j]), by);
            word[j] = *reinterpret_cast<const uint32_t *>(&v);
        }
    } else {
        const float by = mx4_scale_value(scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&halves[j]));
            const __half2 v = __floats2half2_rn(f.x * by, f.y * by);
            word[j] = *reinterpret_cast<const uint32_t *>(&v);
        }
    }
    return make_uint4(word[0], word[1], word[2], word[3]);
}

__device__ __forceinline__ uint4 mx4_put(const uint32_t (&halves)[4], uint32_t scale, __nv_bfloat16)
{
    uint32_t word[4];
    const float by = mx4_scale_value(scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&halves[j]));
        word[j] = cvt_bf16x2_rn(f.y * by, f.x * by);
    }
    return make_uint4(word[0], word[1], word[2], word[3]);
}

__device__ __forceinline__ uint4 mx4_put(const uint32_t (&halves)[4], uint32_t scale, float)
{
    const float by = mx4_scale_value(scale);
    const float2 low = __half22float2(*reinterpret_cast<const __half2 *>(&halves[0]));
    const float2 high = __half22float2(*reinterpret_cast<const __half2 *>(&halves[1]));
    return make_uint4(__float_as_uint(low.x * by), __float_as_uint(low.y * by), __float_as_uint(high.x * by),
                      __float_as_uint(high.y * by));
}

// A lane writes 16 bytes: eight 16-bit values or four floats (28672 x 4096 to binary16 51.5 us, 5.8 TB/s; with twice as much a lane, which
// writes half sectors at a time, 67.1 us).
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
mx4_dequant_kernel(const uint8_t *codes, const uint8_t *scales, uint32_t total_rows, uint32_t k, uint32_t first_row,
                   uint32_t rows, T *__restrict__ out, bool aligned)
{
    constexpr uint32_t kValues = 16u / sizeof(T);
    constexpr uint32_t kLanes = 128u / kValues;          // a chunk
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t row = blockIdx.x * (kQuantThreads / kLanes) + threadIdx.x / kLanes;
    const uint32_t lane = threadIdx.x % kLanes;
    if (row >= rows) {
        return;
    }
    const uint32_t first = blockIdx.y * kQuantChunks;
    const unsigned long long tensor_row = (unsigned long long)first_row + row;
    const uint8_t *code_at = codes + tensor_row * (k / 2u) + first * 64u + lane * (kValues / 2u);
    const uint8_t *scale_at = scales + ((unsigned long long)first * total_rows + tensor_row) * 4u + lane * kValues / 32u;
    T *to = out + (unsigned long long)row * k + first * 128u + lane * kValues;
    uint32_t word[kQuantChunks];
    uint32_t scale[kQuantChunks];
#pragma unroll
    for (uint32_t i = 0; i < kQuantChunks; ++i) {
        if ((first + i) * 128u + lane * kValues < k) {
            word[i] = kValues == 8u ? *reinterpret_cast<const uint32_t *>(code_at + i * 64u)
                                    : (uint32_t)*reinterpret_cast<const uint16_t *>(code_at + i * 64u);
            scale[i] = scale_at[(unsigned long long)i * total_rows * 4u];
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kQuantChunks; ++i) {
        if ((first + i) * 128u + lane * kValues >= k) {
            continue;
        }
        uint32_t halves[4] = {};
        if (kValues == 8u) {
            cvt_f16x2_e2m1(word[i], halves);
        } else {
            cvt_f16x2_e2m1_4((unsigned short)word[i], halves[0], halves[1]);
        }
        const uint4 piece = mx4_put(halves, scale[i], T());
        if (aligned) {
            *reinterpret_cast<uint4 *>(to + i * 128u) = piece;
        } else {
            const T *value = reinterpret_cast<const T *>(&piece);
#pragma unroll
            for (uint32_t j = 0; j < kValues; ++j) {
                to[i * 128u + j] = value[j];
            }
        }
    }
}

static dim3 quant_grid(uint32_t rows, uint32_t rows_a_block, uint32_t k)
{
    return dim3((rows + rows_a_block - 1u) / rows_a_block, (mx4_chunks(k) + kQuantChunks - 1u) / kQuantChunks, 1);
}

cudaError_t launch_mx4_quantize(cudaStream_t stream, bool overlap, const void *x, int x_dtype, uint32_t x_rows,
                                unsigned long long ldx, uint32_t k, const uint32_t *rows_of, uint32_t rows,
                                const uint32_t *rows_dev, void *codes, void *scales, bool own_product)
{
    auto launch = [&](auto kernel, auto *typed) {
        const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15u) == 0u && (ldx * sizeof(*typed)) % 16u == 0u;
        return launch_kernel_early(overlap, kernel, quant_grid(rows, kQuantRows, k), kQuantThreads, 0, stream, typed, x_rows, ldx, k,
                                   rows_of, rows, rows_dev, static_cast<uint2 *>(codes), static_cast<uint8_t *>(scales), aligned);
    };
    auto launch_typed = [&](auto *typed) {
        typedef std::remove_cv_t<std::remove_pointer_t<decltype(typed)>> T;
        return own_product ? launch(mx4_quantize_kernel<T, true>, typed) : launch(mx4_quantize_kernel<T, false>, typed);
    };
    switch (x_dtype) {
    case 0:
        return launch_typed(static_cast<const float *>(x));
    case 1:
        return launch_typed(static_cast<const __half *>(x));
    default:
        return launch_typed(static_cast<const __nv_bfloat16 *>(x));
    }
}

cudaError_t launch_mx4_dequant(cudaStream_t stream, bool overlap, const void *codes, const void *scales,
                               uint32_t total_rows, uint32_t k, uint32_t first_row, uint32_t rows, void *out, int out_dtype)
{
    const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0u;
    auto launch = [&](auto kernel, auto *typed) {
        const uint32_t rows_a_block = kQuantThreads / (128u / (16u / sizeof(*typed)));
        return launch_kernel_early(overlap, kernel, quant_grid(rows, rows_a_block, k), kQuantThreads, 0, stream,
                                   static_cast<const uint8_t *>(codes), static_cast<const uint8_t *>(scales), total_rows, k, first_row, rows, typed, aligned);
    };
    switch (out_dtype) {
    case 0:
        return launch(mx4_dequant_kernel<float>, static_cast<float *>(out));
    case 1:
        return launch(mx4_dequant_kernel<__half>, static_cast<__half *>(out));
    default:
        return launch(mx4_dequant_kernel<__nv_bfloat16>, static_cast<__nv_bfloat16 *>(out));
    }
}

} // namespace q8
