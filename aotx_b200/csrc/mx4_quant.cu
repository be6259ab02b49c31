// Rows of 16- or 32-bit values to MX4 (E2M1 codes, a power of two per 32 values) and back.
//
//   a = max |x_i| over the block,  s = 2^max(floor(log2 a) - 2, -127),  c_i = E2M1(x_i / s), nearest, ties to even
//
// All of it is exact but the last rounding: s is read off the exponent of a, and the division by a power of two is a
// multiplication by another.  Two bytes a value in and half a byte out: memory bounds it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "mx4.h"
#include "mx4_block.cuh"
#include "q8_launch.h"

namespace q8 {

// A lane takes eight values, so 16 lanes a chunk of 128 with its word of four scales, and a warp the same chunk of two
// successive rows; a block 16 rows by kQuantChunks chunks, whose loads are issued together.
constexpr uint32_t kQuantThreads = 256;
constexpr uint32_t kQuantRows = kQuantThreads / 16u;
constexpr uint32_t kQuantChunks = 4;

template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
mx4_quantize_kernel(const T *x, uint32_t x_rows, unsigned long long ldx, uint32_t k, const uint32_t *rows_of, uint32_t rows,
                    const uint32_t *rows_dev, uint32_t *__restrict__ codes, uint32_t *__restrict__ scales, bool aligned)
{
    grid_dependency_wait();
    uint32_t live = rows;
    if (rows_dev != nullptr) {
        const uint32_t on_device = *rows_dev;
        live = on_device < rows ? on_device : rows;
    }
    const uint32_t row = blockIdx.x * kQuantRows + threadIdx.x / 16u;
    const uint32_t lane = threadIdx.x % 16u;
    uint32_t from = row;
    if (row < live && rows_of != nullptr) {
        from = rows_of[row];
    }
    // (all lanes go on: the exchanges below are among whole warps)
    const bool here = row < live && from < x_rows;
    const uint32_t chunks = mx4_chunks(k);
    const T *x_row = x + (here ? (unsigned long long)from * ldx : 0ull);
    for (uint32_t c0 = blockIdx.y * kQuantChunks; c0 < chunks; c0 += gridDim.y * kQuantChunks) {
        Eight<T> raw[kQuantChunks];
        bool in[kQuantChunks];
#pragma unroll
        for (uint32_t i = 0; i < kQuantChunks; ++i) {
            const uint32_t at = (c0 + i) * 128u + lane * 8u;
            in[i] = here && at < k;
            if (in[i]) {
                raw[i].load(x_row + at, aligned);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kQuantChunks; ++i) {
            float v[8] = {};
            if (in[i]) {
                raw[i].floats(v);
            }
            uint32_t largest = mx4_largest(v, 0u);
            largest = max(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 1u));
            largest = max(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 2u));
            const uint32_t scale = mx4_scale(largest);
            const uint32_t word = mx4_codes(v, scale, mx4_inverse(scale));
            if (in[i]) {
                codes[(unsigned long long)row * (k / 8u) + (c0 + i) * 16u + lane] = word;
            }
            // the chunk's four scales, from the first lane of each block, to its first lane; 0 past k
            const uint32_t mine = in[i] ? scale : 0u;
            const uint32_t s1 = __shfl_down_sync(0xFFFFFFFFu, mine, 4u, 16);
            const uint32_t s2 = __shfl_down_sync(0xFFFFFFFFu, mine, 8u, 16);
            const uint32_t s3 = __shfl_down_sync(0xFFFFFFFFu, mine, 12u, 16);
            if (lane == 0u && in[i]) {
                scales[(unsigned long long)(c0 + i) * rows + row] = mine | s1 << 8 | s2 << 16 | s3 << 24;
            }
        }
    }
    // Not before the stores: what is written here may be weights, which a product reads early (aotx_mx4_matmul).
    __syncthreads();
    grid_launch_dependents();
}

// A lane takes eight codes.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
mx4_dequant_kernel(const uint32_t *codes, const uint8_t *scales, uint32_t total_rows, uint32_t k, uint32_t first_row,
                   uint32_t rows, T *__restrict__ out, bool aligned)
{
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t row = blockIdx.x * kQuantRows + threadIdx.x / 16u;
    const uint32_t lane = threadIdx.x % 16u;
    const uint32_t chunks = mx4_chunks(k);
    if (row >= rows) {
        return;
    }
    const unsigned long long tensor_row = (unsigned long long)first_row + row;
    for (uint32_t c0 = blockIdx.y * kQuantChunks; c0 < chunks; c0 += gridDim.y * kQuantChunks) {
        uint32_t word[kQuantChunks];
        uint32_t scale[kQuantChunks];
#pragma unroll
        for (uint32_t i = 0; i < kQuantChunks; ++i) {
            const uint32_t c = c0 + i;
            word[i] = 0u;
            scale[i] = 0u;
            if (c * 128u + lane * 8u < k) {
                word[i] = codes[tensor_row * (k / 8u) + c * 16u + lane];
                scale[i] = scales[((unsigned long long)c * total_rows + tensor_row) * 4u + lane / 4u];
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kQuantChunks; ++i) {
            const uint32_t at = (c0 + i) * 128u + lane * 8u;
            if (at >= k) {
                continue;
            }
            // 2^(scale - 127); the smallest is half of the smallest normal float
            const float by = __uint_as_float(scale[i] == 255u ? 0x7FC00000u : (scale[i] == 0u ? 0x00400000u : scale[i] << 23));
            uint32_t halves[4];
            cvt_f16x2_e2m1(word[i], halves);
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&halves[j]));
                v[2 * j] = f.x * by, v[2 * j + 1] = f.y * by;
            }
            T *to = out + (unsigned long long)row * k + at;
            alignas(16) T rounded[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                store_out<T>(rounded, j, v[j]);
            }
            if (aligned) {
#pragma unroll
                for (uint32_t j = 0; j < sizeof(T) / 2u; ++j) {
                    reinterpret_cast<uint4 *>(to)[j] = reinterpret_cast<const uint4 *>(rounded)[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    to[j] = rounded[j];
                }
            }
        }
    }
}

static dim3 quant_grid(uint32_t rows, uint32_t k)
{
    const uint32_t blocks = (rows + kQuantRows - 1u) / kQuantRows;
    const uint32_t steps = (mx4_chunks(k) + kQuantChunks - 1u) / kQuantChunks;
    return dim3(blocks, steps < 65535u ? steps : 65535u, 1);
}

cudaError_t launch_mx4_quantize(cudaStream_t stream, bool overlap, const void *x, int x_dtype, uint32_t x_rows,
                                unsigned long long ldx, uint32_t k, const uint32_t *rows_of, uint32_t rows,
                                const uint32_t *rows_dev, uint32_t *codes, uint32_t *scales)
{
    auto launch = [&](auto kernel, auto *typed) {
        const bool aligned = (reinterpret_cast<uintptr_t>(x) & 15u) == 0u && (ldx * sizeof(*typed)) % 16u == 0u;
        return launch_kernel_early(overlap, kernel, quant_grid(rows, k), kQuantThreads, 0, stream, typed, x_rows, ldx, k,
                                   rows_of, rows, rows_dev, codes, scales, aligned);
    };
    switch (x_dtype) {
    case 0:
        return launch(mx4_quantize_kernel<float>, static_cast<const float *>(x));
    case 1:
        return launch(mx4_quantize_kernel<__half>, static_cast<const __half *>(x));
    default:
        return launch(mx4_quantize_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16 *>(x));
    }
}

cudaError_t launch_mx4_dequant(cudaStream_t stream, bool overlap, const uint32_t *codes, const uint8_t *scales,
                               uint32_t total_rows, uint32_t k, uint32_t first_row, uint32_t rows, void *out, int out_dtype)
{
    const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15u) == 0u;
    auto launch = [&](auto kernel, auto *typed) {
        return launch_kernel_early(overlap, kernel, quant_grid(rows, k), kQuantThreads, 0, stream, codes, scales, total_rows, k,
                                   first_row, rows, typed, aligned);
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
