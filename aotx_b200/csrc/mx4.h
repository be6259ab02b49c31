// Internal launch interface of the MX4 kernels (mx4_api.cu calls them; the format is described in include/aotx_mx4_b200.h).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "q8_launch.h"

namespace q8 {

constexpr uint32_t kMx4MaxExperts = 256u;

__host__ __device__ inline uint32_t mx4_chunks(uint32_t k)
{
    return (k + 127u) / 128u;   // words of four scales in a row
}

// `own_product`: the launch behind is the product that the quantisation is part of, and may start at once.  Else nothing behind the
// quantisation starts before it has ended.
cudaError_t launch_mx4_quantize(cudaStream_t stream, bool overlap, const void *x, int x_dtype, uint32_t x_rows,
                                unsigned long long ldx, uint32_t k, const uint32_t *rows_of, uint32_t rows,
                                const uint32_t *rows_dev, void *codes, void *scales, bool own_product);
cudaError_t launch_mx4_dequant(cudaStream_t stream, bool overlap, const void *codes, const void *scales,
                               uint32_t total_rows, uint32_t k, uint32_t first_row, uint32_t rows, void *out, int out_dtype);

// A product, or (offsets not null) products grouped by expert.
struct Mx4Product {
    const void *w_codes;
    const uint32_t *w_scales;
    uint32_t experts;          // 1 for a plain product
    uint32_t n, k;
    const void *x_codes;
    const uint32_t *x_scales;
    uint32_t m;                // rows of x
    const uint32_t *m_dev;
    const uint32_t *offsets;
    const uint32_t *y_rows_of;
    uint32_t y_rows;
    void *y;
    int y_dtype;
    unsigned int epilogue;
    bool overlap;
    // x in 16 or 32 bits instead of MX4 (null: x_codes and x_scales), where mx4_linear_quantizes
    const void *x;
    int x_dtype;
    unsigned long long ldx;
};
cudaError_t launch_mx4_product(cudaStream_t stream, const UmmaScratch &scratch, unsigned int sm_count, unsigned int set,
                               const Mx4Product &p);
// Does the product's kernel quantise x itself?
bool mx4_linear_quantizes(uint32_t n, uint32_t k, uint32_t m, unsigned int sm_count);

cudaError_t launch_mx4_order(cudaStream_t stream, bool overlap, const uint32_t *ids, uint32_t tokens,
                             const uint32_t *tokens_dev, uint32_t used, uint32_t experts, uint32_t *order, uint32_t *token_of,
                             uint32_t *offsets);

} // namespace q8
