// Products of MX4 tensors: y[i][j] = sum_c x[i][c] * w[j][c], plain or grouped by expert.
//
// Both operands go to the tensor core as they lie in memory (tcgen05.mma kind::mxf4: E2M1 codes, a power of two per 32
// values of either operand, float sums).  A block takes 128 rows of w, the MMA's rows, by up to 256 rows of x, its columns:
//
//   * Codes come by bulk tensor copies, 256 values (128 bytes) of each row a stage, in the 128-byte swizzle.
//   * Scales come by four warps, a word of four scales (128 values) at a time.  The MMA wants them in tensor memory, row r
//     of the operand in lane r % 32 of column r / 32, the same in each quarter of the lanes: a block of 512 bytes in
//     shared memory, 16 bytes per lane, is laid down so by one tcgen05.cp.  The words of successive rows are neighbours in
//     memory, so rows may start anywhere, as the rows of an expert do.
//   * One thread issues the copies of the scales and the MMAs behind them (they run in that order).  Each stage has its own
//     columns of tensor memory for scales, so that nothing is overwritten before its MMAs are done.
//   * Four warps store: the sums of 16 rows of x are turned round in shared memory, 16 bytes a lane.
#include <cuda.h>

#include "mx4.h"
#include "mx4_ptx.cuh"
#include "q8_rows.cuh"

namespace q8 {

constexpr uint32_t kMxThreads = 320;
constexpr uint32_t kMxScaleWarp = 4;        // the first of four
constexpr uint32_t kMxCopyWarp = 8;
constexpr uint32_t kMxMmaWarp = 9;
constexpr uint32_t kMxRows = 128;           // rows of w per tile
constexpr uint32_t kMxMaxTok = 256;         // rows of x per tile, at most
constexpr uint32_t kMxStageK = 256;         // values of a row per stage
constexpr uint32_t kMxStageBytes = kMxStageK / 2;
constexpr uint32_t kMxMaxStages = 8;
constexpr uint32_t kMxScaleBlock = 512;     // scales of 128 rows and 128 values
constexpr uint32_t kMxAhead = 3;            // stages whose scales are on their way, at most
constexpr uint32_t kMxEpilogueStage = 16u * 32u * 4u;  // per storing warp
constexpr uint32_t kMxBars = 3 * kMxMaxStages + 1;
constexpr uint32_t kMxTail = 4u * kMxEpilogueStage + kMxBars * 8u + 16u;
constexpr uint32_t kMxSmem = 226u * 1024u;

struct MxArgs {
    const uint32_t *w_scales;
    uint32_t w_rows;               // of the tensor, all experts
    const uint32_t *x_scales;
    uint32_t x_rows;
    uint32_t n, k, chunks;
    const uint32_t *m_dev;
    uint32_t experts;
    const uint32_t *offsets;       // grouped, or null
    const uint32_t *y_rows_of;
    uint32_t y_rows;
    void *y;
    uint32_t ldy;
    unsigned int epilogue;
    unsigned int *status;
    uint32_t ntok;                 // rows of x per tile, a multiple of 16
    uint32_t stages, stage_bytes;
    uint32_t tmem_columns;
    uint32_t weights_late;
    uint32_t wide;                 // rows of y lie on 16-byte boundaries
};

__host__ __device__ inline uint32_t mx_scale_blocks(uint32_t ntok)
{
    return ntok > 128u ? 2u : 1u;  // of x, per 128 values
}

// kind::mxf4: both operands E2M1 and K-major, scales powers of two; which half of a word of four scales the MMA's 64 values use.
__host__ __device__ inline uint32_t mx_idesc(uint32_t ntok, uint32_t half)
{
    uint32_t d = 0;
    d |= (2u * half) << 4;         // B's scales: bytes 0, 1 or 2, 3
    d |= 1u << 7;                  // A: E2M1
    d |= 1u << 10;                 // B: E2M1
    d |= (ntok >> 3) << 17;
    d |= 1u << 23;                 // scales: powers of two
    d |= (kMxRows >> 4) << 24;
    d |= (2u * half) << 29;        // A's scales
    return d;
}

// A block of scales in shared memory: rows of 16 bytes, no swizzle, 8 rows (128 bytes) a group.
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t smem_addr)
{
    uint64_t desc = 0;
    desc |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    desc |= (uint64_t)1u << 16;
    desc |= (uint64_t)(128u >> 4) << 32;
    desc |= (uint64_t)1u << 46;
    return desc;
}

// The rows of x of a tile and the expert they belong to; no rows: no tile.
struct MxTile {
    uint32_t expert;
    uint32_t first, rows;
};

// Token tile `index` of the groups in order (all threads call it; `scratch` is shared memory of 33 words).
__device__ __forceinline__ MxTile mx_group_tile(const MxArgs &args, uint32_t index, uint32_t *scratch)
{
    // thread e holds expert e
    const uint32_t e = threadIdx.x;
    uint32_t first = 0u, rows = 0u;
    if (e < args.experts) {
        first = args.offsets[e];
        uint32_t end = args.offsets[e + 1u];
        first = first < args.x_rows ? first : args.x_rows;
        end = end < args.x_rows ? end : args.x_rows;
        rows = end > first ? end - first : 0u;
    }
    const uint32_t tiles = (rows + args.ntok - 1u) / args.ntok;
    uint32_t through = tiles;          // of the experts up to and with this one
#pragma unroll
    for (uint32_t step = 1u; step < 32u; step <<= 1) {
        const uint32_t below = __shfl_up_sync(0xFFFFFFFFu, through, step);
        if ((threadIdx.x & 31u) >= step) {
            through += below;
        }
    }
    if ((threadIdx.x & 31u) == 31u) {
        scratch[threadIdx.x >> 5] = through;
    }
    if (threadIdx.x == 0u) {
        scratch[17] = 0u;              // rows: none
    }
    __syncthreads();
    for (uint32_t w = 0; w < threadIdx.x >> 5; ++w) {
        through += scratch[w];
    }
    if (index < through && index >= through - tiles) {
        const uint32_t skip = (index - (through - tiles)) * args.ntok;
        scratch[16] = first + skip;
        scratch[17] = rows - skip < args.ntok ? rows - skip : args.ntok;
        scratch[18] = e;
    }
    __syncthreads();
    MxTile tile;
    tile.first = scratch[16];
    tile.rows = scratch[17];
    tile.expert = scratch[18];
    return tile;
}

// 16 rows of x (v: this lane's row of w for each) to y, rows `first` and up below `end`.
template <typename YT, bool GATED>
__device__ __forceinline__ void mx_store(const MxArgs &args, uint32_t stage, uint32_t lane, uint32_t first_col, uint32_t columns,
                                         uint32_t first, uint32_t end, const uint32_t (&v)[16])
{
    constexpr uint32_t kColumns = GATED ? 16u : 32u;
    constexpr uint32_t kRowBytes = kColumns * sizeof(YT);
    constexpr uint32_t kLanesPerRow = kColumns / 4u;
    constexpr uint32_t kRowsPerStep = 32u / kLanesPerRow;
    // lane i knows the row of y of row i
    uint32_t row_y = 0xFFFFFFFFu;
    if (lane < 16u && first + lane < end) {
        row_y = args.y_rows_of != nullptr ? args.y_rows_of[first + lane] : first + lane;
        if (row_y >= args.y_rows) {
            row_y = 0xFFFFFFFFu;
        }
    }
    const uint32_t column = GATED ? lane / 2u : lane;
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 16u; ++i) {
        float value = __uint_as_float(v[i]);
        if (GATED) {
            const float other = __shfl_xor_sync(0xFFFFFFFFu, value, 1u);
            value = gated_unit(value, other);
        }
        if (!GATED || (lane & 1u) == 0u) {
            if (sizeof(YT) == 4) {
                st_shared_b32(stage + i * kRowBytes + column * 4u, __float_as_uint(value));
            } else {
                st_shared_b16(stage + i * kRowBytes + column * 2u, out_bits<YT>(value));
            }
        }
    }
    __syncwarp();
    const uint32_t part = lane % kLanesPerRow;
    const bool adds = !GATED && sizeof(YT) == 4 && args.epilogue == kEpilogueAdd;
#pragma unroll
    for (uint32_t step = 0; step < 16u / kRowsPerStep; ++step) {
        const uint32_t local = step * kRowsPerStep + lane / kLanesPerRow;
        const uint32_t row = __shfl_sync(0xFFFFFFFFu, row_y, local);
        const uint32_t from = stage + local * kRowBytes + part * 4u * sizeof(YT);
        if (row == 0xFFFFFFFFu || part * 4u >= columns) {
            continue;
        }
        YT *at = static_cast<YT *>(args.y) + (size_t)row * args.ldy + first_col + part * 4u;
        uint32_t a, b, c = 0u, d = 0u;
        if (sizeof(YT) == 4) {
            ld_shared_v4(from, a, b, c, d);
        } else {
            ld_shared_v2(from, a, b);
        }
        if (args.wide != 0u) {
            if (sizeof(YT) == 4) {
                float4 piece = make_float4(__uint_as_float(a), __uint_as_float(b), __uint_as_float(c), __uint_as_float(d));
                if (adds) {
                    const float4 before = *reinterpret_cast<const float4 *>(at);
                    piece = make_float4(before.x + piece.x, before.y + piece.y, before.z + piece.z, before.w + piece.w);
                }
                *reinterpret_cast<float4 *>(at) = piece;
            } else {
                *reinterpret_cast<uint2 *>(at) = make_uint2(a, b);
            }
        } else {
            const uint32_t words[4] = {a, b, c, d};
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                if (part * 4u + i < columns) {
                    if (sizeof(YT) == 4) {
                        float *cell = reinterpret_cast<float *>(at) + i;
                        const float piece = __uint_as_float(words[i]);
                        *cell = adds ? *cell + piece : piece;
                    } else {
                        reinterpret_cast<unsigned short *>(at)[i] = (unsigned short)(words[i / 2u] >> (16u * (i & 1u)));
                    }
                }
            }
        }
    }
}

template <typename YT, bool GATED>
__global__ void __launch_bounds__(kMxThreads, 1)
mx4_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ MxArgs args)
{
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t scratch[20];
    __shared__ uint32_t abort_flag;
    __shared__ uint32_t tmem_base;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t stages = args.stages;
    const uint32_t x_blocks = mx_scale_blocks(args.ntok);
    // a stage: codes of w, codes of x, scales of w, scales of x
    const uint32_t x_codes_at = kMxRows * kMxStageBytes;
    const uint32_t w_scales_at = x_codes_at + args.ntok * kMxStageBytes;
    const uint32_t x_scales_at = w_scales_at + 2u * kMxScaleBlock;
    const uint32_t tail = base + stages * args.stage_bytes;
    const uint32_t bars = tail + 4u * kMxEpilogueStage;
    auto full = [&](uint32_t s) { return bars + s * 8u; };
    auto scaled = [&](uint32_t s) { return bars + (kMxMaxStages + s) * 8u; };
    auto empty = [&](uint32_t s) { return bars + (2u * kMxMaxStages + s) * 8u; };
    const uint32_t done = bars + 3u * kMxMaxStages * 8u;
    const uint32_t steps = (args.k + kMxStageK - 1u) / kMxStageK;

    if (warp == kMxMmaWarp) {
        tmem_alloc(smem_u32(&tmem_base), args.tmem_columns);
        tmem_relinquish();
    }
    if (threadIdx.x == 0u) {
        abort_flag = 0u;
        for (uint32_t s = 0; s < stages; ++s) {
            mbar_init(full(s), 1u);
            mbar_init(scaled(s), 4u);
            mbar_init(empty(s), 1u);
        }
        mbar_init(done, 1u);
        mbar_init_fence();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_base;

    // which rows
    const uint32_t row0 = blockIdx.x * kMxRows;              // of the expert's n
    MxTile tile = {0u, blockIdx.y * args.ntok, 0u};
    bool early = false;                                      // may the weights come before the work before this has ended?
    if (args.offsets != nullptr) {
        grid_dependency_wait();
        tile = mx_group_tile(args, blockIdx.y, scratch);
    } else if (args.m_dev != nullptr) {
        grid_dependency_wait();
        const uint32_t live = *args.m_dev < args.x_rows ? *args.m_dev : args.x_rows;
        tile.rows = live > tile.first ? (live - tile.first < args.ntok ? live - tile.first : args.ntok) : 0u;
    } else {
        tile.rows = args.x_rows - tile.first < args.ntok ? args.x_rows - tile.first : args.ntok;
        early = args.weights_late == 0u;
    }
    const uint32_t w_row0 = tile.expert * args.n + row0;

    if (tile.rows != 0u) {
        if (warp == kMxCopyWarp) {
            if (elect_one()) {
                const uint32_t bytes = (kMxRows + args.ntok) * kMxStageBytes;
                uint32_t begun = 0;
                if (early) {
                    // weights into every stage, then x behind them
                    begun = steps < stages ? steps : stages;
                    for (uint32_t it = 0; it < begun; ++it) {
                        mbar_expect_tx(full(it), bytes);
                        tma_load_2d(base + it * args.stage_bytes, &map_w, full(it), (int)(it * kMxStageBytes), (int)w_row0);
                    }
                }
                grid_dependency_wait();
                uint32_t it = 0;
                for (; it < steps; ++it) {
                    const uint32_t s = it % stages;
                    const uint32_t at = base + s * args.stage_bytes;
                    if (it >= begun) {
                        if (it >= stages && !mbar_wait(empty(s), (it / stages + 1u) & 1u, &abort_flag, args.status)) {
                            break;
                        }
                        mbar_expect_tx(full(s), bytes);
                        tma_load_2d(at, &map_w, full(s), (int)(it * kMxStageBytes), (int)w_row0);
                    }
                    tma_load_2d(at + x_codes_at, &map_x, full(s), (int)(it * kMxStageBytes), (int)tile.first);
                }
                // No copy is on its way when the block ends, whatever became of the MMAs that wait for them too.
                for (uint32_t last = it > stages ? it - stages : 0u; last < it; ++last) {
                    mbar_wait(full(last % stages), (last / stages) & 1u, &abort_flag, args.status);
                }
            }
        } else if (warp == kMxMmaWarp) {
            if (elect_one()) {
                const uint32_t idesc[2] = {mx_idesc(args.ntok, 0u), mx_idesc(args.ntok, 1u)};
                const uint32_t columns = 2u * 4u * (1u + x_blocks);   // of scales, per stage
                bool ok = true;
                for (uint32_t it = 0; it < steps && ok; ++it) {
                    const uint32_t s = it % stages;
                    const uint32_t parity = (it / stages) & 1u;
                    ok = mbar_wait(scaled(s), parity, &abort_flag, args.status)
                      && mbar_wait(full(s), parity, &abort_flag, args.status);
                    if (!ok) {
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t at = base + s * args.stage_bytes;
                    const uint32_t w_scales = tmem + args.ntok + s * columns;
                    const uint32_t x_scales = w_scales + 8u;
                    for (uint32_t c = 0; c < 2u; ++c) {
                        tmem_copy_scales(w_scales + 4u * c, mx_scale_desc(at + w_scales_at + c * kMxScaleBlock));
                        for (uint32_t b = 0; b < x_blocks; ++b) {
                            tmem_copy_scales(x_scales + 4u * (c * x_blocks + b),
                                             mx_scale_desc(at + x_scales_at + (c * x_blocks + b) * kMxScaleBlock));
                        }
                    }
                    const uint64_t a = umma_desc_sw128(at);
                    const uint64_t b = umma_desc_sw128(at + x_codes_at);
                    const uint32_t left = args.k - it * kMxStageK;
                    const uint32_t pieces = left >= kMxStageK ? 4u : (left + 63u) / 64u;
                    for (uint32_t p = 0; p < pieces; ++p) {
                        // 64 values are 32 bytes of a row
                        umma_mx4(tmem, a + 2u * p, b + 2u * p, idesc[p & 1u], w_scales + 4u * (p >> 1),
                                 x_scales + 4u * x_blocks * (p >> 1), (it | p) != 0u);
                    }
                    umma_commit(empty(s));
                }
                umma_commit(done);
            }
        } else if (warp >= kMxScaleWarp && warp < kMxCopyWarp) {
            // Row t of either operand's tile, and row t + 128 of x.
            grid_dependency_wait();
            const uint32_t t = threadIdx.x - kMxScaleWarp * 32u;
            const uint32_t cell = (t % 32u) * 16u + (t / 32u) * 4u;
            const uint32_t w_row = w_row0 + t;
            const uint32_t ahead = kMxAhead < stages - 1u ? kMxAhead : stages - 1u;
            auto give = [&](uint32_t it) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0u) {
                    mbar_arrive(scaled(it % stages));
                }
            };
            for (uint32_t it = 0; it < steps + ahead; ++it) {
                if (it < steps) {
                    const uint32_t s = it % stages;
                    if (it >= stages && !mbar_wait(empty(s), (it / stages + 1u) & 1u, &abort_flag, args.status)) {
                        break;
                    }
                    const uint32_t at = base + s * args.stage_bytes;
                    for (uint32_t c = 0; c < 2u; ++c) {
                        const uint32_t chunk = 2u * it + c;
                        const bool in = chunk < args.chunks;
                        const bool w_in = in && w_row < args.w_rows;
                        copy_async_4(at + w_scales_at + c * kMxScaleBlock + cell,
                                     args.w_scales + (w_in ? (size_t)chunk * args.w_rows + w_row : 0u), w_in ? 4u : 0u);
                        for (uint32_t b = 0; b < x_blocks; ++b) {
                            const uint32_t r = t + 128u * b;
                            const bool x_in = in && r < tile.rows;
                            copy_async_4(at + x_scales_at + (c * x_blocks + b) * kMxScaleBlock + cell,
                                         args.x_scales + (x_in ? (size_t)chunk * args.x_rows + tile.first + r : 0u),
                                         x_in ? 4u : 0u);
                        }
                    }
                }
                copy_async_commit();
                if (it >= ahead) {
                    // (the groups of the stages after this one may still be on their way)
                    switch (ahead) {
                    case 1u: copy_async_wait<1>(); break;
                    case 2u: copy_async_wait<2>(); break;
                    default: copy_async_wait<3>(); break;
                    }
                    give(it - ahead);
                }
            }
            copy_async_wait_all();
        } else if (warp < kMxScaleWarp) {
            grid_dependency_wait();       // y, and the row map
            if (mbar_wait(done, 0u, &abort_flag, args.status)) {
                tc_fence_after_sync();
                const uint32_t stage = tail + warp * kMxEpilogueStage;
                const uint32_t j0 = row0 + warp * 32u;
                const uint32_t mine = args.n > j0 ? (args.n - j0 < 32u ? args.n - j0 : 32u) : 0u;
                const uint32_t first_col = GATED ? j0 / 2u : j0;
                const uint32_t columns = GATED ? mine / 2u : mine;
                for (uint32_t c0 = 0; c0 < tile.rows; c0 += 16u) {
                    uint32_t v[16];
                    tmem_ld_32x16(tmem + ((warp * 32u) << 16) + c0, v);
                    tmem_ld_wait();
                    mx_store<YT, GATED>(args, stage, lane, first_col, columns, tile.first + c0, tile.first + tile.rows, v);
                }
            }
        }
    }
    // (Behind this block's own wait: what runs early after it then overlaps nothing before it.)
    grid_dependency_wait();
    grid_launch_dependents();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kMxMmaWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, args.tmem_columns);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled()
{
    static const EncodeTiledFn fn = [] {
        void *sym = nullptr;
        cudaDriverEntryPointQueryResult result;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &result) == cudaSuccess
                    && result == cudaDriverEntryPointSuccess
                 ? reinterpret_cast<EncodeTiledFn>(sym) : nullptr;
    }();
    return fn;
}

// Rows of codes, boxes of box_rows rows by one stage, zeros outside.
static bool map_codes(EncodeTiledFn encode, CUtensorMap *map, const void *codes, uint32_t rows, uint32_t k, uint32_t box_rows)
{
    const cuuint64_t dims[2] = {k / 2u, rows};
    const cuuint64_t strides[1] = {k / 2u};
    const cuuint32_t box[2] = {kMxStageBytes, box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
        == CUDA_SUCCESS;
}

static uint32_t up_to(uint32_t v, uint32_t multiple)
{
    return (v + multiple - 1u) / multiple * multiple;
}

template <typename YT>
static cudaError_t launch_typed(cudaStream_t stream, dim3 grid, const CUtensorMap &map_w, const CUtensorMap &map_x,
                                const MxArgs &args, bool overlap)
{
    if (args.epilogue == kEpilogueSwiglu) {
        static unsigned long long configured = 0ull;
        cudaError_t err = allow_shared_memory(mx4_product_kernel<YT, true>, kMxSmem, &configured);
        return err != cudaSuccess ? err
             : launch_kernel_early(overlap, mx4_product_kernel<YT, true>, grid, kMxThreads, kMxSmem, stream, map_w, map_x, args);
    }
    static unsigned long long configured = 0ull;
    cudaError_t err = allow_shared_memory(mx4_product_kernel<YT, false>, kMxSmem, &configured);
    return err != cudaSuccess ? err
         : launch_kernel_early(overlap, mx4_product_kernel<YT, false>, grid, kMxThreads, kMxSmem, stream, map_w, map_x, args);
}

cudaError_t launch_mx4_product(cudaStream_t stream, unsigned int sm_count, const Mx4Product &p)
{
    (void)sm_count;
    const EncodeTiledFn encode = encode_tiled();
    if (encode == nullptr) {
        return cudaErrorNotSupported;
    }
    MxArgs args = {};
    args.w_scales = p.w_scales;
    args.w_rows = p.experts * p.n;
    args.x_scales = p.x_scales;
    args.x_rows = p.m;
    args.n = p.n;
    args.k = p.k;
    args.chunks = mx4_chunks(p.k);
    args.m_dev = p.m_dev;
    args.experts = p.experts;
    args.offsets = p.offsets;
    args.y_rows_of = p.y_rows_of;
    args.y_rows = p.y_rows;
    args.y = p.y;
    args.ldy = p.epilogue == kEpilogueSwiglu ? p.n / 2u : p.n;
    args.epilogue = p.epilogue;
    args.status = p.status;
    args.weights_late = p.weights_late ? 1u : 0u;
    const uint32_t size = p.y_dtype == 0 ? 4u : 2u;
    args.wide = (reinterpret_cast<uintptr_t>(p.y) & (4u * size - 1u)) == 0u && args.ldy % 4u == 0u;
    // Rows of x per tile: equal parts of at most 256.  By expert, about what one has.
    const uint32_t typical = p.offsets != nullptr ? (p.m + p.experts - 1u) / p.experts : p.m;
    const uint32_t parts = (typical + kMxMaxTok - 1u) / kMxMaxTok;
    args.ntok = up_to((typical + parts - 1u) / parts, 16u);
    const uint32_t tok_tiles = p.offsets != nullptr ? p.m / args.ntok + (p.experts < p.m ? p.experts : p.m)
                                                    : (p.m + args.ntok - 1u) / args.ntok;
    const uint32_t x_blocks = mx_scale_blocks(args.ntok);
    args.stage_bytes = up_to((kMxRows + args.ntok) * kMxStageBytes + 2u * (1u + x_blocks) * kMxScaleBlock, 1024u);
    const uint32_t fit = (kMxSmem - 1024u - kMxTail) / args.stage_bytes;
    args.stages = fit < kMxMaxStages ? fit : kMxMaxStages;
    const uint32_t columns = args.ntok + args.stages * 8u * (1u + x_blocks);
    args.tmem_columns = 32u;
    while (args.tmem_columns < columns) {
        args.tmem_columns *= 2u;
    }
    CUtensorMap map_w, map_x;
    if (!map_codes(encode, &map_w, p.w_codes, args.w_rows, p.k, kMxRows)
        || !map_codes(encode, &map_x, p.x_codes, p.m, p.k, args.ntok)) {
        return cudaErrorInvalidValue;
    }
    const dim3 grid((p.n + kMxRows - 1u) / kMxRows, tok_tiles, 1);
    switch (p.y_dtype) {
    case 0:
        return launch_typed<float>(stream, grid, map_w, map_x, args, p.overlap);
    case 1:
        return launch_typed<__half>(stream, grid, map_w, map_x, args, p.overlap);
    default:
        return launch_typed<__nv_bfloat16>(stream, grid, map_w, map_x, args, p.overlap);
    }
}

} // namespace q8
