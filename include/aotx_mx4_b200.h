/* aotx_mx4_b200 - C ABI of the microscaled 4-bit (MX4) tensors: weights and activations in 4.25 bits a value, which the
 * tensor cores of sm_100a multiply as they are.
 *
 * Beside the Q8_0 path of aotx_q8_b200.h and on its contexts; what that header says about return values, streams, devices,
 * threads and captures holds here.  The block format is MXFP4 of the Open Compute Project's microscaling specification
 * (version 1.0): blocks of 32 values along k share a scale, a power of two.
 *
 * An MX4 tensor of `rows` rows of k values (k a multiple of 32) is two arrays:
 *
 *   codes   uint8 [rows][k / 2]: value 2i of a row in the low four bits of byte i, value 2i + 1 in the high four; a code is a
 *           sign (bit 3), two exponent bits and one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  16-byte aligned.
 *   scales  uint8 [ceil(k / 128)][rows][4]: byte b of (c, r) belongs to values 128c + 32b .. 128c + 32b + 31 of row r and
 *           stands for 2^(byte - 127); 255 is NaN, and so is every value of its block.  Bytes of blocks past k are 0
 *           (anything but 255 does).  4-byte aligned.  (The four scales that 128 values of a row need lie together, and the
 *           words of successive rows do, whatever row a tile of the product starts at.)
 *
 * Limits: k up to 2^24; rows of x up to 2^24 (quantisation and dequantisation: 2^31 - 1, as rows of w); grouped, rows of x
 * times rows of an expert's matrix up to 2^40.
 *
 * The reference has no counterpart: its block types (cuda/model/model.cuh:24-36) all are dequantised to binary16 before
 * they are multiplied.
 */
#ifndef AOTX_MX4_B200_H
#define AOTX_MX4_B200_H

#include "aotx_q8_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of x (F32, F16 or BF16, row i at x + i * ldx values, ldx >= k) to MX4.  Output row i, for i < rows, is row i of x or,
 * where rows_of is not null, row rows_of[i]; an entry of rows_of that is not below x_rows names no row, and that output row
 * stays as it is.  (x_rows: how many rows x has; without rows_of, rows <= x_rows.)  rows_dev, if not null, is a device
 * word with the live number of rows: min(*rows_dev, rows) are written; `rows` stays the extent of codes and scales.
 *
 * The scale of a block is 2^(floor(log2 a) - 2), a the block's largest magnitude, and no smaller than 2^-127 (a block of
 * zeros has that scale); values are divided by it, rounded to the nearest code, ties to the even one, and saturate at 6.
 * A block with an infinity or a NaN gets scale 255 and codes 0: all of it is NaN.
 *
 * What is written may be the weights of the product behind it, on this context or another: no launch behind the quantisation starts
 * before it has ended. */
int aotx_mx4_quantize(aotx_q8_ctx *ctx, void *stream, const void *x, int x_dtype, uint32_t x_rows, uint64_t ldx, uint32_t k,
                      const uint32_t *rows_of, uint32_t rows, const uint32_t *rows_dev, void *codes, void *scales);

/* out[r][c] = value c of row first_row + r, for r < rows, as F32, F16 or BF16, rounded once; out is [rows][k] without gaps.
 * total_rows is the extent of codes and scales; first_row + rows <= total_rows. */
int aotx_mx4_dequant(aotx_q8_ctx *ctx, void *stream, const void *codes, const void *scales, uint32_t total_rows, uint32_t k,
                     uint32_t first_row, uint32_t rows, void *out, int out_dtype);

/* y[i][j] = sum_c x[i][c] * w[j][c], float sums of the values that the two MX4 tensors stand for, for i < m and j < n.  What
 * becomes of a sum (`epilogue`: store, add into a float y, gated unit over interleaved rows of w), y's shape and type and the
 * live batch m_dev are as in aotx_q8_matmul_fused; x has m rows, however many of them live.
 *
 * The weights may be read while the operation before the product on the stream is still running (aotx_q8_set_overlap): nothing but
 * aotx_mx4_quantize may write them just before it. */
int aotx_mx4_matmul(aotx_q8_ctx *ctx, void *stream, const void *w_codes, const void *w_scales, uint32_t n, uint32_t k,
                    const void *x_codes, const void *x_scales, uint32_t m, const uint32_t *m_dev, void *y, int y_dtype,
                    int epilogue);

/* aotx_mx4_quantize of x, then aotx_mx4_matmul: the same products, whose float sums may be formed in another order.  Few rows
 * are quantised by the kernel that multiplies them; otherwise `workspace` (16-byte aligned device memory of
 * aotx_mx4_linear_workspace_bytes; 0 where none is needed) holds x in MX4 between the two.  (The weights may be read early
 * here as there: before x is quantised.) */
size_t aotx_mx4_linear_workspace_bytes(const aotx_q8_ctx *ctx, uint32_t n, uint32_t k, uint32_t m);
int aotx_mx4_linear(aotx_q8_ctx *ctx, void *stream, const void *w_codes, const void *w_scales, uint32_t n, uint32_t k,
                    const void *x, int x_dtype, uint64_t ldx, uint32_t m, const uint32_t *m_dev, void *y, int y_dtype,
                    int epilogue, void *workspace, size_t workspace_bytes);

/* The order of the (token, rank) pairs by expert: ids is [tokens][used], as aotx_q8_moe_route leaves it, pair p = token * used +
 * rank.  Pairs of expert e take places offsets[e] .. offsets[e + 1] in ascending order of p; order[place] = p and, where
 * token_of is not null, token_of[place] = p / used.  offsets has experts + 1 entries.  A selection that is not below `experts`
 * names no expert and gets no place; the places left over at the end hold 0xFFFFFFFF.  tokens_dev as in
 * aotx_q8_moe_route: pairs of tokens past it get no place either.  experts <= 256, tokens * used < 2^31. */
int aotx_mx4_moe_order(aotx_q8_ctx *ctx, void *stream, const uint32_t *ids, uint32_t tokens, const uint32_t *tokens_dev,
                       uint32_t used, uint32_t experts, uint32_t *order, uint32_t *token_of, uint32_t *offsets);

/* Products grouped by expert: rows offsets[e] .. offsets[e + 1] of x (`rows` rows, sorted by expert) times expert e's matrix,
 * rows e * n .. e * n + n of w (experts * n rows).  offsets: experts + 1 device words, ascending; an expert may have no
 * row.  Entries past `rows` count as `rows`, and a range that runs backwards as empty.  Row i of the result goes to row i of y or,
 * where y_rows_of is not null, to row y_rows_of[i]; y has y_rows rows, and a row past them is left out (a row that two
 * entries name holds either's result, a value at a time).  Rows of x that no expert has, and their rows of y, are not
 * touched.  epilogue: STORE or SWIGLU (n counts gate and up rows).  experts <= 256. */
int aotx_mx4_matmul_grouped(aotx_q8_ctx *ctx, void *stream, const void *w_codes, const void *w_scales, uint32_t experts,
                            uint32_t n, uint32_t k, const void *x_codes, const void *x_scales, uint32_t rows,
                            const uint32_t *offsets, const uint32_t *y_rows_of, uint32_t y_rows, void *y, int y_dtype,
                            int epilogue);

#ifdef __cplusplus
}
#endif

#endif
