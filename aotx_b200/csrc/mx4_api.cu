// The C ABI of the MX4 tensors: argument checks and the way from a call to its kernels.  Declarations in
// include/aotx_mx4_b200.h.
#include "../../include/aotx_mx4_b200.h"

#include <cuda_runtime.h>

#include "mx4.h"
#include "q8_context.h"

namespace {

const uint32_t kMaxRows = 1u << 24;    // of x; (1 << 31) - 1 of w
const uint32_t kMaxDepth = 1u << 24;
const uint64_t kMaxProducts = 1ull << 40;  // rows of x by an expert's rows of w: the kernel counts its tiles in 32 bits

int fail(aotx_q8_ctx *ctx, cudaError_t err)
{
    ctx->last_cuda = (int)err;
    return AOTX_Q8_ERR_CUDA;
}

int code_of(aotx_q8_ctx *ctx, cudaError_t err)
{
    return err == cudaSuccess ? AOTX_Q8_OK : fail(ctx, err);
}

bool known(int dtype)
{
    return dtype == AOTX_Q8_F32 || dtype == AOTX_Q8_F16 || dtype == AOTX_Q8_BF16;
}

uintptr_t size_of(int dtype)
{
    return dtype == AOTX_Q8_F32 ? 4u : 2u;
}

bool aligned(const void *p, uintptr_t to)
{
    return (reinterpret_cast<uintptr_t>(p) & (to - 1u)) == 0u;
}

bool tensor(const void *codes, const void *scales)
{
    return codes != nullptr && scales != nullptr && aligned(codes, 16u) && aligned(scales, 4u);
}

bool depth(uint32_t k)
{
    return k != 0u && k % 32u == 0u && k <= kMaxDepth;
}

// The context's device is current until the call returns.
struct OnDevice {
    int before = -1;
    int ours;
    explicit OnDevice(const aotx_q8_ctx *ctx) : ours(ctx->device)
    {
        cudaGetDevice(&before);
        if (before != ours) {
            cudaSetDevice(ours);
        }
    }
    ~OnDevice()
    {
        if (before >= 0 && before != ours) {
            cudaSetDevice(before);
        }
    }
};

size_t code_bytes(uint64_t rows, uint32_t k)
{
    return (size_t)rows * (k / 2u);
}

size_t scale_bytes(uint64_t rows, uint32_t k)
{
    return (size_t)rows * q8::mx4_chunks(k) * 4u;
}

bool epilogue_known(int epilogue, uint32_t n, int y_dtype, bool may_add)
{
    return epilogue == AOTX_Q8_EPILOGUE_STORE || (epilogue == AOTX_Q8_EPILOGUE_SWIGLU && n % 2u == 0u)
        || (epilogue == AOTX_Q8_EPILOGUE_ADD && may_add && y_dtype == AOTX_Q8_F32);
}

} // namespace

extern "C" int aotx_mx4_quantize(aotx_q8_ctx *ctx, void *stream, const void *x, int x_dtype, uint32_t x_rows, uint64_t ldx,
                                 uint32_t k, const uint32_t *rows_of, uint32_t rows, const uint32_t *rows_dev, void *codes,
                                 void *scales)
{
    if (ctx == nullptr || !known(x_dtype) || !depth(k) || ldx < k || rows > 0x7FFFFFFFu
        || (rows_of == nullptr && rows > x_rows)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    if (rows == 0u || x_rows == 0u) {
        return AOTX_Q8_OK;
    }
    if (x == nullptr || !aligned(x, size_of(x_dtype)) || !tensor(codes, scales) || !aligned(rows_of, 4u)
        || !aligned(rows_dev, 4u)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    const OnDevice on(ctx);
    return code_of(ctx, q8::launch_mx4_quantize((cudaStream_t)stream, ctx->overlap != 0, x, x_dtype, x_rows, ldx, k, rows_of,
                                                rows, rows_dev, codes, scales, false));
}

extern "C" int aotx_mx4_dequant(aotx_q8_ctx *ctx, void *stream, const void *codes, const void *scales, uint32_t total_rows,
                                uint32_t k, uint32_t first_row, uint32_t rows, void *out, int out_dtype)
{
    if (ctx == nullptr || !known(out_dtype) || !depth(k) || total_rows > 0x7FFFFFFFu || rows > total_rows
        || first_row > total_rows - rows) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    if (rows == 0u) {
        return AOTX_Q8_OK;
    }
    if (!tensor(codes, scales) || out == nullptr || !aligned(out, size_of(out_dtype))) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    const OnDevice on(ctx);
    return code_of(ctx, q8::launch_mx4_dequant((cudaStream_t)stream, ctx->overlap != 0, codes, scales, total_rows, k, first_row, rows,
                                               out, out_dtype));
}

extern "C" int aotx_mx4_matmul(aotx_q8_ctx *ctx, void *stream, const void *w_codes, const void *w_scales, uint32_t n, uint32_t k,
                               const void *x_codes, const void *x_scales, uint32_t m, const uint32_t *m_dev, void *y,
                               int y_dtype, int epilogue)
{
    if (ctx == nullptr || !known(y_dtype) || !depth(k) || n > 0x7FFFFFFFu || m > kMaxRows
        || !epilogue_known(epilogue, n, y_dtype, true)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    if (n == 0u || m == 0u) {
        return AOTX_Q8_OK;
    }
    if (!tensor(w_codes, w_scales) || !tensor(x_codes, x_scales) || y == nullptr || !aligned(y, size_of(y_dtype))
        || !aligned(m_dev, 4u)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    const OnDevice on(ctx);
    q8::Mx4Product p = {};
    p.w_codes = w_codes;
    p.w_scales = static_cast<const uint32_t *>(w_scales);
    p.experts = 1u;
    p.n = n;
    p.k = k;
    p.x_codes = x_codes;
    p.x_scales = static_cast<const uint32_t *>(x_scales);
    p.m = m;
    p.m_dev = m_dev;
    p.y_rows = m;
    p.y = y;
    p.y_dtype = y_dtype;
    p.epilogue = (unsigned int)epilogue;
    p.overlap = ctx->overlap != 0;
    return code_of(ctx, q8::launch_mx4_product((cudaStream_t)stream, ctx->scratch, ctx->sm_count, ctx->launches++, p));
}

extern "C" size_t aotx_mx4_linear_workspace_bytes(const aotx_q8_ctx *ctx, uint32_t n, uint32_t k, uint32_t m)
{
    if (ctx == nullptr || !depth(k) || n == 0u || m == 0u || q8::mx4_linear_quantizes(n, k, m, ctx->sm_count)) {
        return 0u;
    }
    return (code_bytes(m, k) + 255u) / 256u * 256u + scale_bytes(m, k);
}

extern "C" int aotx_mx4_linear(aotx_q8_ctx *ctx, void *stream, const void *w_codes, const void *w_scales, uint32_t n, uint32_t k,
                               const void *x, int x_dtype, uint64_t ldx, uint32_t m, const uint32_t *m_dev, void *y, int y_dtype,
                               int epilogue, void *workspace, size_t workspace_bytes)
{
    if (ctx == nullptr || !known(x_dtype) || !known(y_dtype) || !depth(k) || ldx < k || n > 0x7FFFFFFFu || m > kMaxRows
        || !epilogue_known(epilogue, n, y_dtype, true)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    if (n == 0u || m == 0u) {
        return AOTX_Q8_OK;
    }
    if (!tensor(w_codes, w_scales) || x == nullptr || !aligned(x, size_of(x_dtype)) || y == nullptr
        || !aligned(y, size_of(y_dtype)) || !aligned(m_dev, 4u)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    const size_t need = aotx_mx4_linear_workspace_bytes(ctx, n, k, m);
    if (need != 0u) {
        if (workspace == nullptr || !aligned(workspace, 16u) || workspace_bytes < need) {
            return AOTX_Q8_ERR_WORKSPACE;
        }
        unsigned char *codes = static_cast<unsigned char *>(workspace);
        unsigned char *scales = codes + (code_bytes(m, k) + 255u) / 256u * 256u;
        const OnDevice on(ctx);
        const cudaError_t err = q8::launch_mx4_quantize((cudaStream_t)stream, ctx->overlap != 0, x, x_dtype, m, ldx, k, nullptr, m,
                                                        m_dev, codes, scales, true);
        return err != cudaSuccess ? fail(ctx, err)
             : aotx_mx4_matmul(ctx, stream, w_codes, w_scales, n, k, codes, scales, m, m_dev, y, y_dtype, epilogue);
    }
    const OnDevice on(ctx);
    q8::Mx4Product p = {};
    p.w_codes = w_codes;
    p.w_scales = static_cast<const uint32_t *>(w_scales);
    p.experts = 1u;
    p.n = n;
    p.k = k;
    p.m = m;
    p.m_dev = m_dev;
    p.y_rows = m;
    p.y = y;
    p.y_dtype = y_dtype;
    p.epilogue = (unsigned int)epilogue;
    p.overlap = ctx->overlap != 0;
    p.x = x;
    p.x_dtype = x_dtype;
    p.ldx = ldx;
    return code_of(ctx, q8::launch_mx4_product((cudaStream_t)stream, ctx->scratch, ctx->sm_count, ctx->launches++, p));
}

extern "C" int aotx_mx4_moe_order(aotx_q8_ctx *ctx, void *stream, const uint32_t *ids, uint32_t tokens,
                                  const uint32_t *tokens_dev, uint32_t used, uint32_t experts, uint32_t *order,
                                  uint32_t *token_of, uint32_t *offsets)
{
    if (ctx == nullptr || experts == 0u || experts > q8::kMx4MaxExperts || used == 0u
        || (unsigned long long)tokens * used >= (1ull << 31) || offsets == nullptr || !aligned(offsets, 4u)
        || !aligned(ids, 4u) || !aligned(order, 4u) || !aligned(token_of, 4u) || !aligned(tokens_dev, 4u)
        || (tokens != 0u && (ids == nullptr || order == nullptr))) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    const OnDevice on(ctx);
    return code_of(ctx, q8::launch_mx4_order((cudaStream_t)stream, ctx->overlap != 0, ids, tokens, tokens_dev, used, experts,
                                             order, token_of, offsets));
}

extern "C" int aotx_mx4_matmul_grouped(aotx_q8_ctx *ctx, void *stream, const void *w_codes, const void *w_scales,
                                       uint32_t experts, uint32_t n, uint32_t k, const void *x_codes, const void *x_scales,
                                       uint32_t rows, const uint32_t *offsets, const uint32_t *y_rows_of, uint32_t y_rows,
                                       void *y, int y_dtype, int epilogue)
{
    if (ctx == nullptr || !known(y_dtype) || !depth(k) || experts == 0u || experts > q8::kMx4MaxExperts
        || (unsigned long long)experts * n > 0x7FFFFFFFull || rows > kMaxRows || (uint64_t)rows * n > kMaxProducts
        || !epilogue_known(epilogue, n, y_dtype, false)) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    if (n == 0u || rows == 0u || y_rows == 0u) {
        return AOTX_Q8_OK;
    }
    if (!tensor(w_codes, w_scales) || !tensor(x_codes, x_scales) || offsets == nullptr || !aligned(offsets, 4u)
        || !aligned(y_rows_of, 4u) || y == nullptr || !aligned(y, size_of(y_dtype))) {
        return AOTX_Q8_ERR_ARGUMENT;
    }
    const OnDevice on(ctx);
    q8::Mx4Product p = {};
    p.w_codes = w_codes;
    p.w_scales = static_cast<const uint32_t *>(w_scales);
    p.experts = experts;
    p.n = n;
    p.k = k;
    p.x_codes = x_codes;
    p.x_scales = static_cast<const uint32_t *>(x_scales);
    p.m = rows;
    p.offsets = offsets;
    p.y_rows_of = y_rows_of;
    p.y_rows = y_rows;
    p.y = y;
    p.y_dtype = y_dtype;
    p.epilogue = (unsigned int)epilogue;
    p.overlap = ctx->overlap != 0;
    return code_of(ctx, q8::launch_mx4_product((cudaStream_t)stream, ctx->scratch, ctx->sm_count, ctx->launches++, p));
}
