// Products of MX4 tensors: y[i][j] = sum_c x[i][c] * w[j][c], plain or grouped by expert.
//
// Both operands go to the tensor core as they lie in memory (tcgen05.mma kind::mxf4: E2M1 codes, a power of two per 32
// values of either operand, float sums).  A tile is 128 rows of w, the MMA's rows, by up to 256 rows of x, its columns; a step
// is 256 values of its depth:
//
//   * Codes come by bulk tensor copies, 128 bytes of each row a step, in the 128-byte swizzle.
//   * Scales come by four warps, a word of four scales (128 values) at a time.  The MMA wants them in tensor memory, row r
//     of the operand in lane r % 32 of column r / 32, the same in each quarter of the lanes: a block of 512 bytes in
//     shared memory, 16 bytes per lane, is laid down so by one tcgen05.cp.  The words of successive rows are neighbours in
//     memory, so rows may start anywhere, as the rows of an expert do.
//   * One thread issues the copies of the scales and the MMAs behind them (they run in that order).  Each stage has its own
//     columns of tensor memory for scales, so that nothing is overwritten before its MMAs are done.
//   * Four or eight warps store: the sums of 16 rows of x are turned round in shared memory, 16 bytes a lane.
//   * Few rows of x in 16 or 32 bits (mx4_linear) are quantised by the storing warps, which have nothing else to do at first,
//     straight into the shared memory that the MMA reads, every stage that the block needs once.
//
// Few rows of x are bound by w's bytes, and what a launch costs by itself; many by the way of the codes from L2 to shared memory (with
// all MMAs but a step's first left out, 28672 x 4096 by 2048 rows takes 8 % less).  The forms of the kernel and the ways of dealing
// the steps of all tiles to blocks follow from that:
//
//   * Few tiles: a cluster of 2, 4 or 8 blocks shares one.  Each has a part of its depth; each column's sums go through distributed
//     shared memory to the block that adds them and stores it.  (1024 x 4096 by 8 rows 4.5 us, a block a tile 7.1 us; 8192 x 4096 7.6
//     and 8.4.)
//   * At most a tile a block: blocks have one each.  Rows of x are cut into as many parts as fill the SMs so (8192 x 4096 by 256 rows
//     10.1 us, in one part and equal runs 16.8; 18432 x 4096 by 200 rows 13.0, in equal runs 19.8).
//   * Else blocks have the same number of whole tiles, one behind the other, so copies go on from tile to tile.  What is left over goes
//     to some of them, or is dealt to all as equal runs of steps, before their whole tiles.  A tile that is cut between blocks
//     belongs to the one with its first step: the others leave their sums in the context's scratch and raise a flag per warp (a
//     block does so once, with its first tile, before it waits for anyone), and the owner adds them in the order of the
//     blocks.  (14336 x 8192 by 300 rows 25.0 us; with the cuts behind the whole tiles, where nothing hides their stores, 27.8.)
//   * Two blocks to an SM for few rows of x: one's stores overlap the other's copies.
//   * A pair of blocks on neighbouring SMs for many: 256 rows of w, each block with its 128 and half of x's rows, so that each code is
//     read into shared memory half as often.
#include <cuda.h>

#include "mx4.h"
#include "mx4_block.cuh"
#include "mx4_ptx.cuh"
#include "q8_rows.cuh"

namespace q8 {

// The forms of the kernel: a block to an SM, two, or a pair of blocks on neighbouring SMs that work on one tile.
enum MxForm { kMxOne, kMxTwo, kMxPair };
// Warps of a block: those that store, four that bring scales, one that copies codes, one that issues MMAs.  Two storing warps for each
// quarter of tensor memory's lanes, which take its columns in turn; one where there are few columns.
__host__ __device__ constexpr uint32_t mx_store_warps(MxForm form)
{
    return form == kMxTwo ? 4u : 8u;
}
__host__ __device__ constexpr uint32_t mx_threads(MxForm form)
{
    return (mx_store_warps(form) + 6u) * 32u;
}
constexpr uint32_t kMxRows = 128;           // rows of w per tile
constexpr uint32_t kMxMaxTok = 256;         // rows of x per tile, at most
constexpr uint32_t kMxStageK = 256;         // values of a row per part of a stage: 128 bytes, a row of the swizzle
constexpr uint32_t kMxStageBytes = kMxStageK / 2;
constexpr uint32_t kMxMaxStages = 12;
constexpr uint32_t kMxMaxScales = 16;       // stages whose scales are on their way
constexpr uint32_t kMxMaxSlots = 9;         // stages of x that stay
constexpr uint32_t kMxScaleBlock = 512;     // scales of 128 rows and 128 values
constexpr uint32_t kMxEpilogueStage = 16u * 32u * 4u;  // per storing warp
// Tiles are dealt whole where what the blocks then lose, waiting for those with one more, is no more than this depth on average; cutting
// costs as much.  (36864 x 2048 by 300 rows 17.6 us, with tiles cut 21.8; 19456 x 2560 15.5 and 16.6; 128 experts of 2048 x 768, 4096 pairs,
// 28.7 and 32.9.  By 4096 instead: 28672 x 8192 by 128 rows 28.9, not 27.2; by 2048: 14336 x 4096 by 512 rows 22.7, not 21.5.)
constexpr uint32_t kMxCutDepth = 3000;
// A run is cut from a tile only if it has as many steps.  (With 4, 28672 x 4096 by 300 rows takes 31.1 us, not 28.3, and 20480 x 8192 by 128
// rows 31.0, not 22.5; with 12, 40960 x 4096 by 8 rows 20.6, not 18.8.)
constexpr uint32_t kMxFewSteps = 8;
// Rows of x per tile of a pair of blocks, at most: two accumulators beside the scales.  (28672 x 4096 by 300 rows 30.3 us, with 128
// 34.4; by 2048 rows 118 and 132.)
constexpr uint32_t kMxPairTok = 192;
// Rows of x that pairs take, at least.  (40960 x 2048 by 72 rows 12.1 us, single blocks 13.3, by 128 rows 13.3 and 14.9; 28672 x 4096 by
// 128 rows 16.9 and 17.2, by 2048 rows 118 and 144; by 48 rows 15.7 and 14.0.  128 experts of 1536 x 2048 with 96 rows each 55 and 64.)
constexpr uint32_t kMxPairFrom = 65;
// Rows of x per tile where two blocks share an SM, at most.  (28672 x 4096 by 8 rows 13.4 us, a block to an SM 14.5; by 64 rows 15.0 and
// 15.7; 20480 x 2048 by 48 rows 7.5 and 9.4; but 40960 x 4096 by 64 rows, cut, 23.5 and 21.0, and 65536 x 4096 by 96 rows 34.3 and 31.7.)
constexpr uint32_t kMxTwoTok = 64;
// And where they are a cluster's.  (18432 x 4096 by 1 row 10.7 us, a block to an SM 12.0; by 64 rows 13.3 and 11.1.)
constexpr uint32_t kMxTwoClusterTok = 32;
// Tiles of a product that is multiplied by clusters, at most: as many clusters of each size as the GPU runs at the same time, twice as
// many where two blocks share an SM.  (More wait for the first to end: 4096 x 8192 by 1 row, 32 tiles, by eights 8.5 us, by fours
// 7.9; 12288 x 4096, 96 tiles, by twos with a block to an SM 15.4, with two blocks 8.6.)
constexpr uint32_t kMxClustersOf8 = 12;
constexpr uint32_t kMxClustersOf4 = 32;
constexpr uint32_t kMxClustersOf2 = 72;
// Steps of a block of a larger cluster, at least (2 or 3: the same; with 6, 1024 x 4096 by 1 row takes 6.8 us, not 4.9).
constexpr uint32_t kMxClusterSteps = 4;
// Steps of a tile that a cluster of two shares, at least: up to kMxTwoClusterTok rows of x per tile, and more.  (Time by clusters and with
// a block a tile: 8192 x 1024 by 8 rows 4.7 and 4.2 us, x 2048, in 16 bits, 1 row 5.9 and 6.1; x 1024 by 64 rows 6.6 and 4.7, x 2560 7.6 and
// 6.6, x 4096 8.7 both.)
constexpr uint32_t kMxClusterSteps2 = 7;
constexpr uint32_t kMxClusterSteps2Wide = 14;
// And rows of x per tile, at most.  Narrower tiles come first where there are clusters for all: less to exchange (512 x 2048 by 128 rows
// in one part 7.3 us, in two 5.5, in four 4.7; 6144 x 4096 by 100 rows in one part by clusters 9.4, in two, a block each, 8.7; 8192 x 2048
// by 128 rows 6.8 and 6.6; but 6144 x 8192 by 100 rows 12.8 and 13.9).
constexpr uint32_t kMxClusterTok = 64;
// What the kernel quantises of x itself: few rows, and few stages of them.  Every block turns the stages that it needs by itself; a
// launch of its own costs a microsecond more than the product alone.  4096 x 4096 (4 stages a block), 1 row, 6.4 us against 7.3 apart, 8
// rows 6.9 against 7.4, 16 rows 9.2 against 7.5; 12288 x 4096 (8 stages), 4 rows, 8.8 against 9.3, 8 rows 10.6 against 9.3; 20000 x 4096
// (9 stages), 2 rows, 12.4 against 12.9, 8 rows 14.1 against 12.9.
constexpr uint32_t kMxFusedRows = 16;
constexpr uint32_t kMxFusedWork = 32;       // rows times stages
constexpr uint32_t kMxBars = 2 * kMxMaxStages + 5 + kMxMaxSlots + 2 * kMxMaxScales;
__host__ __device__ constexpr uint32_t mx_smem(MxForm form)
{
    return (form == kMxTwo ? 109u : 223u) * 1024u;
}
// Shared memory for stages and what stays, the first part; the rest is the storing warps' and the barriers.
__host__ __device__ constexpr uint32_t mx_rings(MxForm form)
{
    return (mx_smem(form) - 1024u - mx_store_warps(form) * kMxEpilogueStage - kMxBars * 8u) / 1024u * 1024u;
}

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
    uint32_t stages, stage_bytes;  // of codes
    uint32_t scale_slots, scale_bytes;
    uint32_t tmem_columns, accumulators;
    uint32_t scale_places;         // stages whose scales are in tensor memory at a time
    uint32_t wide;                 // rows of y lie on 16-byte boundaries
    // x in 16 or 32 bits, quantised here: its stages stay in `slots` places behind the ring
    const void *x;
    uint32_t x_type;
    uint32_t x_aligned;
    unsigned long long ldx;
    uint32_t slots;                // 0: x is in MX4 and goes through the ring
    uint32_t cluster;              // blocks that share a tile; 0: each has whole tiles, and runs of those left over or a whole one more
    uint32_t share;                // columns of the tile that a block of the cluster adds up and stores
    float *partial;                // per block: [row of x][row of w], and its flags
    unsigned int *flags;
    unsigned long long tile_floats;
};

// Parts of a stage.  A wait, a commit and what else the thread that issues the MMAs does for a stage take it as long as four MMAs of
// 208 columns: pairs of blocks have two parts to a stage (28672 x 4096 by 2048 rows 118 us, with one 129).  A single block has one,
// so that few steps can be dealt evenly.
__host__ __device__ constexpr uint32_t mx_parts(MxForm form)
{
    return form == kMxPair ? 2u : 1u;
}

__host__ __device__ inline uint32_t mx_scale_blocks(uint32_t ntok)
{
    return ntok > 128u ? 2u : 1u;  // of x, per 128 values
}

// kind::mxf4: both operands E2M1 and K-major, scales powers of two; which half of a word of four scales the MMA's 64 values use.
__host__ __device__ inline uint32_t mx_idesc(uint32_t rows, uint32_t ntok, uint32_t half)
{
    uint32_t d = 0;
    d |= (2u * half) << 4;         // B's scales: bytes 0, 1 or 2, 3
    d |= 1u << 7;                  // A: E2M1
    d |= 1u << 10;                 // B: E2M1
    d |= (ntok >> 3) << 17;
    d |= 1u << 23;                 // scales: powers of two
    d |= (rows >> 4) << 24;
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

// The groups of a grouped product, in shared memory: expert e's rows of x from first[e], rows[e] of them, and the tiles up
// to and with it.
struct MxGroups {
    uint32_t first[kMx4MaxExperts];
    uint32_t rows[kMx4MaxExperts];
    uint32_t through[kMx4MaxExperts];
    uint32_t warps[8];
};

// Every thread calls it, once the offsets are there.  Returns the number of tiles.
__device__ __forceinline__ uint32_t mx_groups(const MxArgs &args, MxGroups &groups, uint32_t row_tiles)
{
    const uint32_t e = threadIdx.x;
    uint32_t through = 0u;
    if (e < kMx4MaxExperts) {
        uint32_t first = 0u, rows = 0u;
        if (e < args.experts) {
            first = args.offsets[e];
            uint32_t end = args.offsets[e + 1u];
            first = first < args.x_rows ? first : args.x_rows;
            end = end < args.x_rows ? end : args.x_rows;
            rows = end > first ? end - first : 0u;
        }
        through = (rows + args.ntok - 1u) / args.ntok * row_tiles;
#pragma unroll
        for (uint32_t step = 1u; step < 32u; step <<= 1) {
            const uint32_t below = __shfl_up_sync(0xFFFFFFFFu, through, step);
            if ((threadIdx.x & 31u) >= step) {
                through += below;
            }
        }
        groups.first[e] = first;
        groups.rows[e] = rows;
        if ((threadIdx.x & 31u) == 31u) {
            groups.warps[e / 32u] = through;
        }
    }
    __syncthreads();
    if (e < kMx4MaxExperts) {
        for (uint32_t w = 0; w < e / 32u; ++w) {
            through += groups.warps[w];
        }
        groups.through[e] = through;
    }
    __syncthreads();
    return groups.through[kMx4MaxExperts - 1u];
}

// A tile: 128 rows of w (256 of a pair of blocks) from w_row (row `row0` of n), and rows of x.
struct MxTile {
    uint32_t w_row, row0;
    uint32_t first, rows;
};

// Finds the tiles of a run one after the other; the tiles of one run of rows of w follow each other, so that the second finds
// it in L2.
struct MxTiles {
    uint32_t expert = 0, begin = 0, end = 0;     // of tiles of the expert that the last one belonged to
    uint32_t tok_tiles = 0;
    uint32_t row_tile = 0, tok_tile = 0;         // the next one
    uint32_t following = 0xFFFFFFFFu;            // its index

    __device__ __forceinline__ MxTile next(const MxArgs &args, const MxGroups &groups, uint32_t tile_rows, uint32_t index,
                                           uint32_t all_tok_tiles, uint32_t live)
    {
        if (index != following) {
            uint32_t in = index;
            tok_tiles = all_tok_tiles;
            end = 0xFFFFFFFFu;
            if (args.offsets != nullptr) {
                // the expert is the first whose tiles go past the index
                uint32_t low = 0u, high = args.experts - 1u;
                while (low < high) {
                    const uint32_t middle = (low + high) / 2u;
                    if (groups.through[middle] > index) {
                        high = middle;
                    } else {
                        low = middle + 1u;
                    }
                }
                expert = low;
                begin = expert != 0u ? groups.through[expert - 1u] : 0u;
                end = groups.through[expert];
                tok_tiles = (groups.rows[expert] + args.ntok - 1u) / args.ntok;
                in -= begin;
            }
            row_tile = in / tok_tiles;
            tok_tile = in - row_tile * tok_tiles;
        } else if (index == end) {
            // the next expert that has tiles
            do {
                ++expert;
                end = groups.through[expert];
            } while (end == index);
            tok_tiles = (groups.rows[expert] + args.ntok - 1u) / args.ntok;
            row_tile = 0u;
            tok_tile = 0u;
        }
        following = index + 1u;
        const uint32_t first = args.offsets != nullptr ? groups.first[expert] : 0u;
        const uint32_t rows = args.offsets != nullptr ? groups.rows[expert] : live;
        const uint32_t skip = tok_tile * args.ntok;
        MxTile tile;
        tile.row0 = row_tile * tile_rows;
        tile.w_row = expert * args.n + tile.row0;
        tile.first = first + skip;
        tile.rows = rows > skip ? (rows - skip < args.ntok ? rows - skip : args.ntok) : 0u;
        if (++tok_tile == tok_tiles) {
            tok_tile = 0u;
            ++row_tile;
        }
        return tile;
    }
};

// The run of steps of block b: of `units` in all, the first units % blocks blocks take one more.
__host__ __device__ __forceinline__ unsigned long long mx_run_begin(uint32_t b, uint32_t blocks, unsigned long long units)
{
    const unsigned long long share = units / blocks;
    const unsigned long long more = units - share * blocks;
    return b * share + (b < more ? b : more);
}

// Workers that `units` steps are enough for: a run is shorter than a tile's depth only if it is kMxFewSteps parts of 256 values or
// more, because cutting a tile costs as much as several steps.
__host__ __device__ __forceinline__ unsigned long long mx_workers(unsigned long long units, uint32_t steps, uint32_t parts)
{
    const uint32_t few = steps < kMxFewSteps / parts ? steps : kMxFewSteps / parts;
    const unsigned long long workers = units / few;
    return workers != 0ull ? workers : 1ull;
}

// The pieces of a run, and of whole tiles behind it: a tile and the steps [from, to) of its depth.
struct MxPieces {
    uint32_t left;                 // steps of the run that no piece has had
    uint32_t then_tile, then_left; // and of the tiles behind it
    uint32_t steps;
    uint32_t tile, from, to;
    bool begun;

    __device__ __forceinline__ void set(unsigned long long unit, unsigned long long end, uint32_t depth)
    {
        left = (uint32_t)(end - unit);
        steps = depth;
        tile = unit != 0ull ? (uint32_t)(unit / depth) : 0u;
        from = (uint32_t)(unit - (unsigned long long)tile * depth);
        to = from;
        begun = false;
        then_left = 0u;
    }

    __device__ __forceinline__ void then(uint32_t first, uint32_t tiles)
    {
        then_tile = first;
        then_left = tiles * steps;
    }

    __device__ __forceinline__ bool next()
    {
        if (left == 0u) {
            if (then_left == 0u) {
                return false;
            }
            left = then_left;
            then_left = 0u;
            tile = then_tile;
            from = 0u;
            begun = false;
        }
        if (begun) {
            ++tile;
            from = 0u;
        }
        begun = true;
        to = left < steps - from ? from + left : steps;
        left -= to - from;
        return true;
    }
};

// A place in a ring of stages, and how often the ring has come round, as the parity that its barriers are waited for with.
struct MxRing {
    uint32_t at = 0, parity = 0;

    __device__ __forceinline__ void next(uint32_t size)
    {
        if (++at == size) {
            at = 0;
            parity ^= 1u;
        }
    }
};

// Has the block that this flag belongs to left its sums?  Bounded like every wait.
__device__ __forceinline__ bool mx_wait_flag(const unsigned int *flag, volatile uint32_t *abort_flag, unsigned int *status)
{
    const long long begin = clock64();
    while (ld_acquire_gpu(flag) == 0u) {
        if (*abort_flag != 0u || clock64() - begin > Q8_WAIT_CYCLES) {
            *abort_flag = 1u;
            atomicOr(status, Q8_DEV_FLAG_TIMEOUT);
            return false;
        }
    }
    return true;
}

// The stages of x that this block needs, in the order in which it needs them, by the storing warps: a warp takes a row of a
// stage, 8 values a lane and four lanes a block of 32, the loads of several such rows together.  A warp arrives on a stage's
// barrier when its rows of it are there.  (The places hold zeros before: rows past the last, values past k.)
template <typename T, uint32_t WARPS>
__device__ __forceinline__ void mx_quantize_x(const MxArgs &args, const T *x, uint32_t place, uint32_t slot_bytes,
                                              uint32_t bars, uint32_t first_step, uint32_t slots, uint32_t steps, uint32_t live)
{
    constexpr uint32_t kTogether = 2u;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t block = lane / 4u;
    // the next row of the next stage, for the loads and for the stores
    uint32_t slot = 0u, row = warp;
    uint32_t told = 0u;                    // stages whose barrier this warp has arrived on
    while (row >= live && slot < slots) {
        row -= live;
        ++slot;
        if (live == 0u) {
            slot = slots;
        }
    }
    while (slot < slots) {
        Eight<T> raw[kTogether];
        uint32_t cell[kTogether], scale_at[kTogether];
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j) {
            cell[j] = 0u;
            raw[j].zero();
            if (slot < slots) {
                const uint32_t step = first_step + slot < steps ? first_step + slot : first_step + slot - steps;
                const uint32_t at = step * kMxStageK + lane * 8u;
                const uint32_t stage = place + slot * slot_bytes;
                if (at < args.k) {
                    cell[j] = stage + row * kMxStageBytes + ((block ^ (row & 7u)) * 16u) + (lane & 3u) * 4u;
                    raw[j].load(x + (unsigned long long)row * args.ldx + at, args.x_aligned != 0u);
                }
                scale_at[j] = stage + args.ntok * kMxStageBytes + (block / 4u) * kMxScaleBlock + (row % 32u) * 16u + block % 4u;
                row += WARPS;
                while (row >= live) {
                    row -= live;
                    ++slot;
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j) {
            uint32_t largest = Eight<T>::largest(raw[j], raw[j]);
            largest = max(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 1u));
            largest = max(largest, __shfl_xor_sync(0xFFFFFFFFu, largest, 2u));
            const uint32_t scale = mx4_scale(largest);
            const uint32_t word = raw[j].codes(scale, mx4_inverse(scale));
            if (cell[j] != 0u) {
                st_shared_b32(cell[j], word);
                if ((lane & 3u) == 0u) {
                    st_shared_b8(scale_at[j], scale);
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        for (; told < slot && told < slots; ++told) {
            if (lane == 0u) {
                mbar_arrive(bars + told * 8u);
            }
        }
    }
    fence_proxy_async_smem();
    __syncwarp();
    for (; told < slots; ++told) {
        if (lane == 0u) {
            mbar_arrive(bars + told * 8u);
        }
    }
}

// silu(gate) * up.  For a float y as the Q8_0 products form it; for 16 bits by the approximate exponential and reciprocal, which are
// off by 2^-18 of the result at most for gates from -14 on, and by 2^-16 down to -88, against 2^-11 and 2^-8 of the rounding: 6
// instructions instead of 20 (28672 x 4096 by 2048 rows 119 us, with the exact unit 137; by 8 rows 13.9 and 14.0).  Below -88.73 the
// exponential is infinite and the result a zero with its sign, in either form, as gate / (1 + expf(-gate)) is in floats.
template <typename YT>
__device__ __forceinline__ float mx_gated(float gate, float up)
{
    if (sizeof(YT) == 4) {
        return gated_unit(gate, up);
    }
    return gate * rcp_approx(1.0f + ex2_approx(gate * -1.4426950408889634f)) * up;
}

// Where a storing warp's columns of a tile go in y, as one of its lanes needs it: `y` is at the lane's 16 bytes of row 0 (wide) or at
// its column.
template <typename YT>
struct MxOut {
    YT *y;
    uint32_t ldy;
    bool in;                       // the lane has columns of the tile
    bool wide, adds;
};

template <typename YT, bool GATED>
__device__ __forceinline__ MxOut<YT> mx_out(const MxArgs &args, uint32_t lane, uint32_t first_col, uint32_t columns)
{
    constexpr uint32_t kPiece = 16u / sizeof(YT);
    constexpr uint32_t kLanesPerRow = (GATED ? 16u : 32u) / kPiece;
    MxOut<YT> out;
    out.ldy = args.ldy;
    out.wide = args.wide != 0u;
    out.adds = !GATED && sizeof(YT) == 4 && args.epilogue == kEpilogueAdd;
    const uint32_t column = out.wide ? lane % kLanesPerRow * kPiece : lane;
    out.in = column < columns;
    out.y = static_cast<YT *>(args.y) + first_col + column;
    return out;
}

// 16 rows of x (v: this lane's row of w for each) to y; lane i's row_y is the row of y of row i, 0xFFFFFFFF for none.  They are
// turned round in the warp's own shared memory and written 16 bytes a lane.  GATED: neighbouring lanes hold gate
// and up of a column (arithmetic of cuda/model/norm.cu:92-105); of two rows of x the even lane forms the first's value and
// the odd lane the second's.
template <typename YT, bool GATED>
__device__ __forceinline__ void mx_store(const MxOut<YT> &out, uint32_t stage, uint32_t lane, uint32_t row_y, const uint32_t (&v)[16])
{
    constexpr uint32_t kRowBytes = (GATED ? 16u : 32u) * sizeof(YT);
    constexpr uint32_t kLanesPerRow = kRowBytes / 16u;
    constexpr uint32_t kRowsPerStep = 32u / kLanesPerRow;
    constexpr uint32_t kSteps = 16u / kRowsPerStep;
    // (the rows that this lane writes are known before anything is waited for)
    uint32_t row[kSteps];
#pragma unroll
    for (uint32_t step = 0; step < kSteps; ++step) {
        row[step] = __shfl_sync(0xFFFFFFFFu, row_y, step * kRowsPerStep + lane / kLanesPerRow);
    }
    auto put = [&](uint32_t at_row, uint32_t column, float value) {
        if (sizeof(YT) == 4) {
            st_shared_b32(stage + at_row * kRowBytes + column * 4u, __float_as_uint(value));
        } else {
            st_shared_b16(stage + at_row * kRowBytes + column * 2u, out_bits<YT>(value));
        }
    };
    __syncwarp();                  // the rows before these are out of it
    if (GATED) {
        const bool odd = (lane & 1u) != 0u;
        float got[8], value[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            got[i] = __shfl_xor_sync(0xFFFFFFFFu, __uint_as_float(odd ? v[2u * i] : v[2u * i + 1u]), 1u);
        }
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            const float keep = __uint_as_float(odd ? v[2u * i + 1u] : v[2u * i]);
            value[i] = mx_gated<YT>(odd ? got[i] : keep, odd ? keep : got[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            put(2u * i + (odd ? 1u : 0u), lane / 2u, value[i]);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16u; ++i) {
            put(i, lane, __uint_as_float(v[i]));
        }
    }
    __syncwarp();
    if (out.wide) {
        uint4 piece[kSteps];
#pragma unroll
        for (uint32_t step = 0; step < kSteps; ++step) {
            ld_shared_v4(stage + step * 512u + lane * 16u, piece[step].x, piece[step].y, piece[step].z, piece[step].w);
        }
        if (out.adds) {
            float4 before[kSteps];
#pragma unroll
            for (uint32_t step = 0; step < kSteps; ++step) {
                before[step] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (out.in && row[step] != 0xFFFFFFFFu) {
                    before[step] = *reinterpret_cast<const float4 *>(out.y + (size_t)row[step] * out.ldy);
                }
            }
#pragma unroll
            for (uint32_t step = 0; step < kSteps; ++step) {
                piece[step].x = __float_as_uint(before[step].x + __uint_as_float(piece[step].x));
                piece[step].y = __float_as_uint(before[step].y + __uint_as_float(piece[step].y));
                piece[step].z = __float_as_uint(before[step].z + __uint_as_float(piece[step].z));
                piece[step].w = __float_as_uint(before[step].w + __uint_as_float(piece[step].w));
            }
        }
#pragma unroll
        for (uint32_t step = 0; step < kSteps; ++step) {
            if (out.in && row[step] != 0xFFFFFFFFu) {
                *reinterpret_cast<uint4 *>(out.y + (size_t)row[step] * out.ldy) = piece[step];
            }
        }
    } else {
        // rows of y off the boundary: a value a lane
#pragma unroll 4
        for (uint32_t i = 0; i < 16u; ++i) {
            const uint32_t to = __shfl_sync(0xFFFFFFFFu, row_y, i);
            if (to == 0xFFFFFFFFu || !out.in) {
                continue;
            }
            YT *at = out.y + (size_t)to * out.ldy;
            if (sizeof(YT) == 4) {
                const float value = ld_shared_f32(stage + i * kRowBytes + lane * 4u);
                *reinterpret_cast<float *>(at) = out.adds ? *reinterpret_cast<float *>(at) + value : value;
            } else {
                *reinterpret_cast<unsigned short *>(at) = ld_shared_u16(stage + i * kRowBytes + lane * 2u);
            }
        }
    }
}

// What another block left of 16 rows of x by this lane's row of w: four rows of x side by side, [row of x / 4][row of w][row of x % 4].
__device__ __forceinline__ void mx_fetch_partial(float4 (&part)[4], const float4 *slot)
{
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        part[i] = __ldcg(slot + i * kMxRows);
    }
}

__device__ __forceinline__ void mx_add_partial(uint32_t (&v)[16], const float4 (&part)[4])
{
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        v[4u * i] = __float_as_uint(__uint_as_float(v[4u * i]) + part[i].x);
        v[4u * i + 1u] = __float_as_uint(__uint_as_float(v[4u * i + 1u]) + part[i].y);
        v[4u * i + 2u] = __float_as_uint(__uint_as_float(v[4u * i + 2u]) + part[i].z);
        v[4u * i + 3u] = __float_as_uint(__uint_as_float(v[4u * i + 3u]) + part[i].w);
    }
}

// Columns of a tile of `rows` rows of x that block `rank` of a cluster adds up (columns change hands by fours).
__device__ __forceinline__ uint32_t mx_share(const MxArgs &args, uint32_t rank, uint32_t rows)
{
    const uint32_t first = rank * args.share;
    const uint32_t all = (rows + 3u) & ~3u;
    const uint32_t left = all > first ? all - first : 0u;
    return left < args.share ? left : args.share;
}

template <typename YT, bool GATED, MxForm FORM>
__global__ void __launch_bounds__(mx_threads(FORM), FORM == kMxTwo ? 2 : 1)
mx4_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ MxArgs args)
{
    constexpr bool PAIR = FORM == kMxPair;
    constexpr uint32_t kStoreWarps = mx_store_warps(FORM);
    constexpr uint32_t kScaleWarp = kStoreWarps;
    constexpr uint32_t kCopyWarp = kStoreWarps + 4u;
    constexpr uint32_t kMmaWarp = kStoreWarps + 5u;
    extern __shared__ unsigned char smem_raw[];
    __shared__ MxGroups groups;
    __shared__ uint32_t abort_flag;
    __shared__ uint32_t tmem_base;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t stages = args.stages;
    const uint32_t x_blocks = mx_scale_blocks(args.ntok);
    const bool stays = !PAIR && args.slots != 0u;
    const bool clusters = !PAIR && args.cluster != 0u;
    // a pair of blocks is one worker: each has half of the tile's rows of w, its sums, and half of its rows of x
    constexpr uint32_t kBlocks = PAIR ? 2u : 1u;
    constexpr uint32_t kParts = mx_parts(FORM);
    constexpr uint32_t kStepK = kParts * kMxStageK;
    constexpr uint32_t kTileRows = kBlocks * kMxRows;
    const uint32_t half = PAIR ? cluster_ctarank() : 0u;
    const uint32_t worker = PAIR ? blockIdx.x / 2u : blockIdx.x;
    uint32_t workers = PAIR ? gridDim.x / 2u : gridDim.x;
    const uint32_t x_rows = PAIR ? args.ntok / 2u : args.ntok;     // of a tile, in this block's shared memory
    // A stage: codes of w, codes of x; its scales, of w and of x, lie behind all stages.  They come by other copies than the codes and
    // take longer: of a pair, which has room for few stages, they have a ring and barriers of their own and more of them are on their
    // way (28672 x 4096, 2048 rows, 116.9 -> 113.0 us; a single block loses by it, 4096 x 4096, 1 row, 6.3 -> 6.5 us: another wait a
    // stage).  x that stays has places behind both.
    constexpr bool kApart = PAIR;
    const uint32_t x_codes_at = kParts * kMxRows * kMxStageBytes;
    const uint32_t scales = base + stages * args.stage_bytes;
    const uint32_t scale_slots = args.scale_slots;
    const uint32_t x_scales_at = 2u * kParts * kMxScaleBlock;
    const uint32_t place = scales + scale_slots * args.scale_bytes;
    const uint32_t slot_bytes = args.ntok * kMxStageBytes + 2u * x_blocks * kMxScaleBlock;
    const uint32_t tail = base + mx_rings(FORM);
    const uint32_t bars = tail + kStoreWarps * kMxEpilogueStage;
    auto full = [&](uint32_t s) { return bars + s * 8u; };           // codes are there, and scales that are not apart
    auto empty = [&](uint32_t s) { return bars + (kMxMaxStages + s) * 8u; };
    auto summed = [&](uint32_t b) { return bars + (2u * kMxMaxStages + b) * 8u; };
    auto taken = [&](uint32_t b) { return bars + (2u * kMxMaxStages + 2u + b) * 8u; };
    const uint32_t exchanged = bars + (2u * kMxMaxStages + 4u) * 8u;
    const uint32_t x_bars = bars + (2u * kMxMaxStages + 5u) * 8u;
    auto scaled = [&](uint32_t s) { return kApart ? bars + (kMxBars - 2u * kMxMaxScales + s) * 8u : full(s); };
    auto used = [&](uint32_t s) { return kApart ? bars + (kMxBars - kMxMaxScales + s) * 8u : empty(s); };
    // a cluster's exchange: per block of it this block's columns, [block][four columns][row of w][column] floats, at the end of the rings
    const uint32_t exchange = tail - (clusters ? args.cluster * args.share * kMxRows * 4u : 0u);
    const uint32_t rank = clusters ? blockIdx.x % args.cluster : 0u;

    if (warp == kMmaWarp) {
        if (PAIR) {
            pair_tmem_alloc(smem_u32(&tmem_base), args.tmem_columns);
            pair_tmem_relinquish();
        } else {
            tmem_alloc(smem_u32(&tmem_base), args.tmem_columns);
            tmem_relinquish();
        }
    }
    // A barrier a thread: one after the other they take a microsecond of the smallest launches.
    if (threadIdx.x < kMxBars) {
        const uint32_t i = threadIdx.x;
        uint32_t count = kStoreWarps;                          // taken, and the stages of x that stay
        if (!kApart && i < kMxMaxStages) {
            count = 1u + 128u;
        } else if (i < 2u * kMxMaxStages + 2u || i == 2u * kMxMaxStages + 4u || i >= kMxBars - kMxMaxScales) {
            count = 1u;                                          // full, empty, summed, exchanged, used
        } else if (i >= kMxBars - 2u * kMxMaxScales) {
            count = half == 0u ? 128u + 1u : 128u;               // the second block of a pair tells the first of its scales
        } else if (PAIR && i < 2u * kMxMaxStages + 4u) {
            count = 2u * kStoreWarps;
        }
        mbar_init(bars + i * 8u, count);
        mbar_init_fence();
        if (clusters && i == 2u * kMxMaxStages + 4u) {
            const uint32_t tok_tiles = (args.x_rows + args.ntok - 1u) / args.ntok;
            const uint32_t skip = blockIdx.x / args.cluster % tok_tiles * args.ntok;
            const uint32_t rows = args.x_rows - skip < args.ntok ? args.x_rows - skip : args.ntok;
            mbar_expect_tx(exchanged, mx_share(args, rank, rows) * kMxRows * 4u * args.cluster);
        }
    }
    if (threadIdx.x == 0u) {
        abort_flag = 0u;
    }
    if (PAIR || clusters) {
        // every block of the cluster has started, and its barriers count, before another block reaches into it
        __syncwarp();
        cluster_arrive_release();
    }
    if (stays && warp < kStoreWarps) {
        for (uint32_t at = threadIdx.x * 16u; at < args.slots * slot_bytes; at += kStoreWarps * 32u * 16u) {
            st_shared_v4(place + at, 0u, 0u, 0u, 0u);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (PAIR) {
        __syncwarp();
        cluster_wait_acquire();
    }
    tc_fence_after_sync();
    const uint32_t tmem = tmem_base;

    // which tiles there are
    const uint32_t steps = (args.k + kStepK - 1u) / kStepK;
    const uint32_t row_tiles = (args.n + kTileRows - 1u) / kTileRows;
    uint32_t live = args.x_rows;
    uint32_t tok_tiles = (args.x_rows + args.ntok - 1u) / args.ntok;
    uint32_t tiles = tok_tiles * row_tiles;
    bool waited = false;                   // has everything before this launch ended?
    if (args.offsets != nullptr) {
        grid_dependency_wait();
        waited = true;
        tiles = mx_groups(args, groups, row_tiles);
    } else if (args.m_dev != nullptr && tok_tiles > 1u) {
        grid_dependency_wait();
        waited = true;
        live = *args.m_dev < args.x_rows ? *args.m_dev : args.x_rows;
        tok_tiles = (live + args.ntok - 1u) / args.ntok;
        tiles = tok_tiles * row_tiles;
    }
    const bool early = !waited;            // weights may come before that
    // Each block has `each` whole tiles; those left over go whole to the first blocks, where what the others then lose is less than
    // cutting tiles costs, or are cut: dealt in runs of steps, which come before a block's whole tiles, so that what cutting adds to
    // the stores is behind their copies.  (x that stays is quantised for one run: all tiles are cut then.)
    const uint32_t each = stays ? 0u : tiles / workers;
    const uint32_t over = tiles - each * workers;
    const bool whole = !stays && (over == 0u || (unsigned long long)(workers - over) * args.k <= (unsigned long long)kMxCutDepth * workers);
    const unsigned long long units = whole ? 0ull : (unsigned long long)over * steps;
    MxPieces mine;
    mine.set(0ull, 0ull, steps);
    if (clusters) {
        const unsigned long long first = (unsigned long long)(blockIdx.x / args.cluster) * steps;
        mine.set(first + mx_run_begin(rank, args.cluster, steps), first + mx_run_begin(rank + 1u, args.cluster, steps), steps);
    } else if (whole) {
        mine.then(worker * each + (worker < over ? worker : over), each + (worker < over ? 1u : 0u));
    } else {
        // (the device may know of fewer tiles than the launch provided for)
        const uint32_t cutters = workers;
        const unsigned long long enough = mx_workers(units, steps, kParts);
        workers = enough < cutters ? (uint32_t)enough : cutters;
        if (worker < workers) {
            mine.set(mx_run_begin(worker, workers, units), mx_run_begin(worker + 1u, workers, units), steps);
        }
        mine.then(over + worker * each, each);
    }
    const uint32_t run = mine.left;
    const uint32_t first_step = mine.from;
    MxTiles finder;
    auto tile_at = [&](MxTiles &tiles_found, uint32_t index) {
        return tiles_found.next(args, groups, kTileRows, index, tok_tiles, live);
    };
    // (a batch of one tile is multiplied whole, however much of it lives)
    const auto live_rows = [&]() {
        if (args.m_dev != nullptr && tok_tiles == 1u && !waited) {
            const uint32_t on_device = *args.m_dev;
            return on_device < args.x_rows ? on_device : args.x_rows;
        }
        return live;
    };

    if (warp == kCopyWarp) {
        if (elect_one()) {
            // (a pair's codes all count on the first block's barrier, which that block arms for both)
            const uint32_t bytes = kParts * (kMxRows + (stays ? 0u : x_rows)) * kMxStageBytes;
            const uint32_t signal = PAIR ? mapa_shared(bars, 0u) : bars;
            auto copy = [&](uint32_t to, const CUtensorMap *map, uint32_t s, uint32_t step, uint32_t row, uint32_t rows) {
#pragma unroll
                for (uint32_t part = 0; part < kParts; ++part) {
                    const int from = (int)((step * kParts + part) * kMxStageBytes);
                    if (PAIR) {
                        pair_tma_load_2d(to + part * rows * kMxStageBytes, map, signal + s * 8u, from, (int)row);
                    } else {
                        tma_load_2d(to + part * rows * kMxStageBytes, map, signal + s * 8u, from, (int)row);
                    }
                }
            };
            auto copy_w = [&](uint32_t s, uint32_t step, uint32_t w_row) {
                if (!PAIR || half == 0u) {
                    mbar_expect_tx(full(s), PAIR ? 2u * bytes : bytes);
                }
                copy(base + s * args.stage_bytes, &map_w, s, step, w_row + half * kMxRows, kMxRows);
            };
            uint32_t begun = 0;
            if (early) {
                // weights into every stage, then x behind them
                MxPieces ahead = mine;
                MxTiles found;
                while (begun < stages && ahead.next()) {
                    const MxTile tile = tile_at(found, ahead.tile);
                    for (uint32_t step = ahead.from; step < ahead.to && begun < stages; ++step) {
                        copy_w(begun++, step, tile.w_row);
                    }
                }
            }
            if (!stays || !early) {
                grid_dependency_wait();
            }
            uint32_t it = 0;
            MxRing ring;
            bool ok = true;
            while (ok && mine.next()) {
                const MxTile tile = tile_at(finder, mine.tile);
                for (uint32_t step = mine.from; step < mine.to; ++step, ++it, ring.next(stages)) {
                    if (it >= begun) {
                        if (it >= stages && !mbar_wait_hot(empty(ring.at), ring.parity ^ 1u, &abort_flag, args.status)) {
                            ok = false;
                            break;
                        }
                        copy_w(ring.at, step, tile.w_row);
                    }
                    if (!stays) {
                        copy(base + ring.at * args.stage_bytes + x_codes_at, &map_x, ring.at, step, tile.first + half * x_rows, x_rows);
                    }
                }
            }
            // Everything is on its way: the blocks of the next launch may take their places as these leave them.  (Behind this
            // block's own wait, so that what runs early overlaps nothing before it.)
            grid_dependency_wait();
            grid_launch_dependents();
            // No copy is on its way when the block ends, whatever became of the MMAs that wait for them too.
            // (The first block of a pair waits for both; the second stays until the first has seen them.)
            for (uint32_t last = it > stages ? it - stages : 0u; half == 0u && last < it; ++last) {
                mbar_wait(full(last % stages), (last / stages) & 1u, &abort_flag, args.status);
            }
        }
    } else if (PAIR && warp == kMmaWarp && half != 0u) {
        // This block's scales are there: told to the first block, whose thread copies them to tensor memory.
        if (elect_one()) {
            const uint32_t signal = mapa_shared(scaled(0u), 0u);
            MxRing ring;
            bool ok = true;
            while (ok && mine.next()) {
                for (uint32_t step = mine.from; step < mine.to; ++step, ring.next(scale_slots)) {
                    if (!mbar_wait_hot(scaled(ring.at), ring.parity, &abort_flag, args.status)) {
                        ok = false;
                        break;
                    }
                    // (Without release at cluster scope, which takes this thread 1700 cycles: the scales are read from this block's
                    // own shared memory into its own tensor memory, behind the fence.)
                    fence_proxy_async_smem();
                    mbar_arrive_cluster(signal + ring.at * 8u);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        if (elect_one()) {
            const uint32_t idesc0 = mx_idesc(kTileRows, args.ntok, 0u);
            const uint32_t idesc1 = mx_idesc(kTileRows, args.ntok, 1u);
            auto copy_scales = [&](uint32_t to, uint64_t from) {
                if (PAIR) {
                    pair_tmem_copy_scales(to, from);
                } else {
                    tmem_copy_scales(to, from);
                }
            };
            auto multiply = [&](uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t a_scales, uint32_t b_scales,
                                uint32_t accumulate) {
                if (PAIR) {
                    pair_mma_mx4(d, a, b, idesc, a_scales, b_scales, accumulate);
                } else {
                    umma_mx4(d, a, b, idesc, a_scales, b_scales, accumulate);
                }
            };
            auto commit = [&](uint32_t bar) {
                if (PAIR) {
                    pair_commit(bar);
                } else {
                    umma_commit(bar);
                }
            };
            const uint32_t columns = kParts * 8u * (1u + x_blocks);   // of scales, per stage
            const uint32_t scales_at = tmem + args.accumulators * args.ntok;
            const uint64_t codes_desc = umma_desc_sw128(0u);
            const uint64_t scale_desc = mx_scale_desc(0u);
            uint32_t it = 0, piece = 0;
            MxRing ring, slot, sums_ring, scale_place, scale_ring, behind;
            bool ok = true;
            bool ready = false, unused = false, empty_sums = false;
            for (; ok && mine.next(); ++piece, sums_ring.next(args.accumulators)) {
                const uint32_t sums = tmem + sums_ring.at * args.ntok;
                if (piece >= args.accumulators && !empty_sums
                    && !mbar_wait_hot(taken(sums_ring.at), sums_ring.parity ^ 1u, &abort_flag, args.status)) {
                    break;
                }
                for (uint32_t step = mine.from; step < mine.to; ++step, ++it, slot.next(args.slots),
                              scale_place.next(args.scale_places)) {
                    if (!ready && ((stays && it < args.slots && !mbar_wait_hot(x_bars + slot.at * 8u, 0u, &abort_flag, args.status))
                                   || !mbar_wait_hot(full(ring.at), ring.parity, &abort_flag, args.status)
                                   || (kApart && !mbar_wait_hot(scaled(scale_ring.at), scale_ring.parity, &abort_flag, args.status)))) {
                        ok = false;
                        break;
                    }
                    if (PAIR && it >= args.scale_places) {
                        // the scales that lie where these go have been used
                        if (!unused && !mbar_wait_hot(empty(behind.at), behind.parity, &abort_flag, args.status)) {
                            ok = false;
                            break;
                        }
                        behind.next(stages);
                    }
                    // The next stage is asked for now: the answer comes while this one's instructions are issued (a wait takes 200
                    // cycles even where nothing is missing, as much as these).
                    const uint32_t now = ring.at;
                    const uint32_t now_scales = kApart ? scale_ring.at : now;
                    ring.next(stages);
                    scale_ring.next(scale_slots);
                    ready = (!stays || it + 1u >= args.slots)
                        && (!kApart || mbar_test(scaled(scale_ring.at), scale_ring.parity) != 0u)
                        && mbar_test(full(ring.at), ring.parity) != 0u;
                    unused = PAIR && mbar_test(empty(behind.at), behind.parity) != 0u;
                    if (step + 1u == mine.to) {
                        MxRing after = sums_ring;
                        after.next(args.accumulators);
                        empty_sums = mbar_test(taken(after.at), after.parity ^ 1u) != 0u;
                    }
                    tc_fence_after_sync();
                    fence_proxy_async_smem();            // the scales came by ordinary copies
                    const uint32_t at = base + now * args.stage_bytes;
                    const uint32_t x_at = stays ? place + slot.at * slot_bytes : at + x_codes_at;
                    const uint32_t w_scales = scales_at + scale_place.at * columns;
                    const uint32_t x_scales = w_scales + kParts * 8u;
                    const uint32_t scales_from = scales + now_scales * args.scale_bytes;
                    const uint64_t w_from = scale_desc | (scales_from >> 4);
                    const uint64_t x_from = scale_desc | ((stays ? x_at + x_rows * kMxStageBytes : scales_from + x_scales_at) >> 4);
                    // (a block of scales: 128 values of 128 rows)
#pragma unroll
                    for (uint32_t c = 0; c < 2u * kParts; ++c) {
                        copy_scales(w_scales + 4u * c, w_from + c * (kMxScaleBlock >> 4));
                        copy_scales(x_scales + 4u * c, x_from + c * (kMxScaleBlock >> 4));
                    }
                    if (x_blocks == 2u) {
#pragma unroll
                        for (uint32_t c = 2u * kParts; c < 4u * kParts; ++c) {
                            copy_scales(x_scales + 4u * c, x_from + c * (kMxScaleBlock >> 4));
                        }
                    }
                    // 64 values are 32 bytes of a row, and half of a word of scales
                    const uint32_t left = args.k - step * kStepK;
#pragma unroll
                    for (uint32_t p = 0; p < 4u * kParts; ++p) {
                        if (p == 0u || left > 64u * p) {
                            const uint32_t part = p / 4u;
                            multiply(sums, codes_desc | ((at + part * kMxRows * kMxStageBytes) >> 4) + 2u * (p % 4u),
                                     codes_desc | ((x_at + part * x_rows * kMxStageBytes) >> 4) + 2u * (p % 4u),
                                     p % 2u == 0u ? idesc0 : idesc1, w_scales + 4u * (p / 2u), x_scales + 4u * x_blocks * (p / 2u),
                                     p != 0u || step != mine.from);
                        }
                    }
                    commit(empty(now));
                    if (kApart) {
                        commit(used(now_scales));
                    }
                }
                commit(summed(sums_ring.at));
            }
        }
    } else if (warp >= kScaleWarp && warp < kCopyWarp) {
        // Row t of either operand's tile, and row t + 128 of x.
        if (!stays || !early) {
            grid_dependency_wait();
        }
        const uint32_t t = threadIdx.x - kScaleWarp * 32u;
        const uint32_t cell = (t % 32u) * 16u + (t / 32u) * 4u;
        // The copies of as many stages as the ring has are on their way together, and count themselves on the ring's barriers.
        uint32_t it = 0;
        MxRing ring;
        bool ok = true;
        while (ok && mine.next()) {
            const MxTile tile = tile_at(finder, mine.tile);
            const uint32_t w_row = tile.w_row + half * kMxRows + t;
            const bool w_in = w_row < args.w_rows;
            const bool x_in = t < tile.rows;
            const bool x_in_2 = t + 128u < tile.rows;
            // (a row outside the tensor is not read, whatever its address)
            const uint32_t *w_from = args.w_scales + (w_in ? (size_t)(2u * kParts * mine.from) * args.w_rows + w_row : 0u);
            const uint32_t *x_from = stays ? nullptr
                : args.x_scales + (x_in ? (size_t)(2u * kParts * mine.from) * args.x_rows + tile.first + t : 0u);
            for (uint32_t step = mine.from; step < mine.to; ++step, ++it, ring.next(scale_slots)) {
                if (it >= scale_slots && !mbar_wait_hot(used(ring.at), ring.parity ^ 1u, &abort_flag, args.status)) {
                    ok = false;
                    break;
                }
                const uint32_t at = scales + ring.at * args.scale_bytes + cell;
#pragma unroll
                for (uint32_t c = 0; c < 2u * kParts; ++c) {
                    const bool in = 2u * kParts * step + c < args.chunks;
                    copy_async_4(at + c * kMxScaleBlock, w_from, w_in && in ? 4u : 0u);
                    w_from += w_in && in ? args.w_rows : 0u;
                    if (!stays) {
                        copy_async_4(at + x_scales_at + c * x_blocks * kMxScaleBlock, x_from, x_in && in ? 4u : 0u);
                        if (x_blocks == 2u) {
                            copy_async_4(at + x_scales_at + (2u * c + 1u) * kMxScaleBlock, x_in_2 ? x_from + 128u : x_from,
                                         x_in_2 && in ? 4u : 0u);
                        }
                        x_from += x_in && in ? args.x_rows : 0u;
                    }
                }
                copy_async_arrive(scaled(ring.at));
            }
        }
        copy_async_wait_all();
    } else if (warp < kStoreWarps) {
        grid_dependency_wait();       // x, y, the row map and the scratch
        const uint32_t valid = live_rows();
        if (stays) {
            const uint32_t slots = run < args.slots ? run : args.slots;
            switch (args.x_type) {
            case 0u:
                mx_quantize_x<float, kStoreWarps>(args, static_cast<const float *>(args.x), place, slot_bytes, x_bars, first_step,
                    slots, steps, valid);
                break;
            case 1u:
                mx_quantize_x<__half, kStoreWarps>(args, static_cast<const __half *>(args.x), place, slot_bytes, x_bars, first_step,
                    slots, steps, valid);
                break;
            default:
                mx_quantize_x<__nv_bfloat16, kStoreWarps>(args, static_cast<const __nv_bfloat16 *>(args.x), place, slot_bytes, x_bars, first_step,
                    slots, steps, valid);
                break;
            }
        }
        const uint32_t stage = tail + warp * kMxEpilogueStage;
        const uint32_t quarter = (warp & 3u) * 32u;            // this warp's lanes of tensor memory, rows of w
        constexpr uint32_t kTurn = kStoreWarps * 4u;           // its columns, rows of x: 16 of each turn's
        const uint32_t c_first = (warp >> 2) * 16u;
        const uint32_t lane_taddr = tmem + (quarter << 16);
        if (clusters) {
            __syncwarp();
            cluster_wait_acquire();        // the others have started
        }
        const uint32_t signal = PAIR ? mapa_shared(bars, 0u) - bars : 0u;      // from this block's barriers to the first's
        for (MxRing ring; mine.next(); ring.next(args.accumulators)) {
            const MxTile tile = tile_at(finder, mine.tile);
            const uint32_t last_row = tile.first + tile.rows < valid || args.offsets != nullptr ? tile.first + tile.rows : valid;
            // Lane i knows the row of y of row i of 16 of x (fetched before the sums are waited for, and those of the next 16
            // beside the stores of these).
            auto row_of = [&](uint32_t c0) {
                const uint32_t row_x = tile.first + c0 + lane;
                uint32_t row_y = 0xFFFFFFFFu;
                if (lane < 16u && row_x < last_row) {
                    row_y = args.y_rows_of != nullptr ? args.y_rows_of[row_x] : row_x;
                }
                return row_y;
            };
            uint32_t next_row = row_of(c_first);
            // The blocks behind this one that hold the rest of its depth; the first one's sums come while this one's are waited for and
            // stored (a block to an SM: two have no registers for that).
            constexpr bool kAhead = FORM != kMxTwo;
            auto slot_of = [&](uint32_t o) {
                return reinterpret_cast<const float4 *>(args.partial + (blockIdx.x + (1u + o) * kBlocks) * args.tile_floats) + quarter + lane;
            };
            float4 ahead[4];
            uint32_t others = 0u;
            if (!clusters && mine.from == 0u && mine.to < steps) {
                const unsigned long long tile_end = (unsigned long long)(mine.tile + 1u) * steps;
                while (mx_run_begin(worker + others + 1u, workers, units) < tile_end) {
                    ++others;
                }
                bool there = true;
                for (uint32_t o = lane; o < others; o += 32u) {
                    there = there && mx_wait_flag(args.flags + (blockIdx.x + (1u + o) * kBlocks) * kFlagWords + warp, &abort_flag, args.status);
                }
                if (!__all_sync(0xFFFFFFFFu, there)) {
                    break;
                }
                __syncwarp();
                if (kAhead) {
                    mx_fetch_partial(ahead, slot_of(0u) + c_first / 4u * kMxRows);
                }
            }
            if (!mbar_wait_hot(summed(ring.at), ring.parity, &abort_flag, args.status)) {
                break;
            }
            tc_fence_after_sync();
            const uint32_t sums = lane_taddr + ring.at * args.ntok;
            const uint32_t giving = taken(ring.at);
            auto release = [&] {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0u) {
                    if (PAIR) {
                        mbar_arrive_cluster(giving + signal);
                    } else {
                        mbar_arrive(giving);
                    }
                }
            };
            const uint32_t j0 = tile.row0 + half * kMxRows + quarter;
            const uint32_t width = args.n > j0 ? (args.n - j0 < 32u ? args.n - j0 : 32u) : 0u;
            const uint32_t first_col = GATED ? j0 / 2u : j0;
            const MxOut<YT> out = mx_out<YT, GATED>(args, lane, first_col, GATED ? width / 2u : width);
            if (clusters) {
                // One piece per block: each column's sums go to the block of the cluster that adds them up.
                for (uint32_t c0 = c_first; c0 < tile.rows; c0 += kTurn) {
                    uint32_t v[16];
                    tmem_ld_32x16(sums + c0, v);
                    tmem_ld_wait();
                    uint32_t owner = c0 / args.share;
                    uint32_t column = c0 - owner * args.share;
#pragma unroll
                    for (uint32_t i = 0; i < 16u; i += 4u) {
                        if (c0 + i < tile.rows) {
                            const uint32_t to = exchange + ((rank * args.share + column) * kMxRows + (quarter + lane) * 4u) * 4u;
                            store_counted_v4(mapa_shared(to, owner), v[i], v[i + 1u], v[i + 2u], v[i + 3u],
                                             mapa_shared(exchanged, owner));
                        }
                        column += 4u;
                        if (column == args.share) {
                            column = 0u;
                            ++owner;
                        }
                    }
                }
                const uint32_t here = mx_share(args, rank, tile.rows);
                if (here == 0u || !mbar_wait_counted(exchanged, 0u, &abort_flag, args.status)) {
                    break;
                }
                for (uint32_t c0 = c_first; c0 < here; c0 += kTurn) {
                    uint32_t v[16] = {};
                    for (uint32_t r = 0; r < args.cluster; ++r) {
                        const uint32_t from = exchange + ((r * args.share + c0) * kMxRows + (quarter + lane) * 4u) * 4u;
#pragma unroll
                        for (uint32_t i = 0; i < 16u; i += 4u) {
                            if (c0 + i < here) {
                                uint32_t part[4];
                                ld_shared_v4(from + i * kMxRows * 4u, part[0], part[1], part[2], part[3]);
#pragma unroll
                                for (uint32_t j = 0; j < 4u; ++j) {
                                    v[i + j] = r == 0u ? part[j]
                                                       : __float_as_uint(__uint_as_float(v[i + j]) + __uint_as_float(part[j]));
                                }
                            }
                        }
                    }
                    const uint32_t row_x = tile.first + rank * args.share + c0 + lane;
                    const bool stores = lane < 16u && c0 + lane < here && row_x < last_row;
                    mx_store<YT, GATED>(out, stage, lane, stores ? row_x : 0xFFFFFFFFu, v);
                }
                break;
            }
            if (mine.from != 0u) {
                // Another block owns the tile: its sums go to the scratch.
                float4 *left = reinterpret_cast<float4 *>(args.partial + blockIdx.x * args.tile_floats) + quarter + lane;
                for (uint32_t c0 = c_first; c0 < tile.rows; c0 += kTurn) {
                    uint32_t v[16];
                    tmem_ld_32x16(sums + c0, v);
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) {
                        __stcg(left + (c0 / 4u + i) * kMxRows,
                               make_float4(__uint_as_float(v[4u * i]), __uint_as_float(v[4u * i + 1u]),
                                           __uint_as_float(v[4u * i + 2u]), __uint_as_float(v[4u * i + 3u])));
                    }
                }
                release();
                if (lane == 0u) {
                    __threadfence();
                    st_release_gpu(args.flags + blockIdx.x * kFlagWords + warp, 1u);
                }
                continue;
            }
            if (c_first >= tile.rows) {
                release();
            }
            for (uint32_t c0 = c_first; c0 < tile.rows; c0 += kTurn) {
                // (looked at here only: the load has had the last rows' time)
                const uint32_t row_y = next_row < args.y_rows ? next_row : 0xFFFFFFFFu;
                next_row = row_of(c0 + kTurn);
                uint32_t v[16];
                tmem_ld_32x16(sums + c0, v);
                tmem_ld_wait();
                if (c0 + kTurn >= tile.rows) {
                    release();
                }
                if (others != 0u) {
                    if (kAhead) {
                        mx_add_partial(v, ahead);
                    }
#pragma unroll 1
                    for (uint32_t o = kAhead ? 1u : 0u; o < others; ++o) {
                        float4 more[4];
                        mx_fetch_partial(more, slot_of(o) + c0 / 4u * kMxRows);
                        mx_add_partial(v, more);
                    }
                    if (kAhead && c0 + kTurn < tile.rows) {
                        mx_fetch_partial(ahead, slot_of(0u) + (c0 + kTurn) / 4u * kMxRows);
                    }
                }
                mx_store<YT, GATED>(out, stage, lane, row_y, v);
            }
            __syncwarp();
            for (uint32_t o = lane; o < others; o += 32u) {
                args.flags[(blockIdx.x + (1u + o) * kBlocks) * kFlagWords + warp] = 0u;   // for the next launch
            }
        }
    }
    grid_dependency_wait();
    grid_launch_dependents();
    tc_fence_before_sync();
    __syncthreads();
    if (PAIR || clusters) {
        // No block leaves while another of the cluster may reach into it.
        __syncwarp();
        if (clusters && warp >= kStoreWarps) {
            cluster_wait_acquire();
        }
        __syncwarp();
        cluster_arrive_relaxed();
        cluster_wait_acquire();
    }
    if (warp == kMmaWarp) {
        tc_fence_after_sync();
        if (PAIR) {
            pair_tmem_dealloc(tmem, args.tmem_columns);
        } else {
            tmem_dealloc(tmem, args.tmem_columns);
        }
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

template <typename YT, bool GATED, MxForm FORM>
static cudaError_t launch_one(cudaStream_t stream, uint32_t grid, const CUtensorMap &map_w, const CUtensorMap &map_x,
                              const MxArgs &args, bool overlap)
{
    static unsigned long long configured = 0ull;
    const cudaError_t err = allow_shared_memory(mx4_product_kernel<YT, GATED, FORM>, mx_smem(FORM), &configured, FORM == kMxTwo);
    if (err != cudaSuccess) {
        return err;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid, 1, 1);
    config.blockDim = dim3(mx_threads(FORM), 1, 1);
    config.dynamicSmemBytes = mx_smem(FORM);
    config.stream = stream;
    cudaLaunchAttribute attribute[2];
    unsigned int count = 0;
    if (overlap) {
        attribute[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attribute[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    if (FORM == kMxPair || args.cluster > 1u) {
        attribute[count].id = cudaLaunchAttributeClusterDimension;
        attribute[count].val.clusterDim.x = FORM == kMxPair ? 2u : args.cluster;
        attribute[count].val.clusterDim.y = 1;
        attribute[count].val.clusterDim.z = 1;
        ++count;
    }
    config.attrs = attribute;
    config.numAttrs = count;
    return cudaLaunchKernelEx(&config, mx4_product_kernel<YT, GATED, FORM>, map_w, map_x, args);
}

template <typename YT, bool GATED>
static cudaError_t launch_form(cudaStream_t stream, uint32_t grid, MxForm form, const CUtensorMap &map_w,
                               const CUtensorMap &map_x, const MxArgs &args, bool overlap)
{
    switch (form) {
    case kMxOne:
        return launch_one<YT, GATED, kMxOne>(stream, grid, map_w, map_x, args, overlap);
    case kMxTwo:
        return launch_one<YT, GATED, kMxTwo>(stream, grid, map_w, map_x, args, overlap);
    default:
        return launch_one<YT, GATED, kMxPair>(stream, grid, map_w, map_x, args, overlap);
    }
}

template <typename YT>
static cudaError_t launch_typed(cudaStream_t stream, uint32_t grid, MxForm form, const CUtensorMap &map_w,
                                const CUtensorMap &map_x, const MxArgs &args, bool overlap)
{
    return args.epilogue == kEpilogueSwiglu ? launch_form<YT, true>(stream, grid, form, map_w, map_x, args, overlap)
                                            : launch_form<YT, false>(stream, grid, form, map_w, map_x, args, overlap);
}

static uint32_t steps_of(uint32_t k, MxForm form)
{
    return (k + mx_parts(form) * kMxStageK - 1u) / (mx_parts(form) * kMxStageK);
}

static uint32_t row_tiles_of(uint32_t n, MxForm form)
{
    const uint32_t rows = form == kMxPair ? 2u * kMxRows : kMxRows;
    return (n + rows - 1u) / rows;
}

// How a product is multiplied: the form of the kernel, rows of x per tile, and how the steps of its tiles are dealt to blocks.
struct MxPlan {
    MxForm form;
    uint32_t ntok;
    uint32_t cluster;              // blocks that share a tile; 0: whole tiles, those left over whole or in equal runs of steps
    uint32_t grid;
    uint32_t slots;                // stages of x that a block of mx4_linear keeps, 0: x comes in MX4
};

static void deal(MxPlan &plan, unsigned long long tiles, uint32_t steps, uint32_t workers)
{
    const unsigned long long enough = mx_workers(tiles * steps, steps, mx_parts(plan.form));
    plan.cluster = 0u;
    plan.grid = enough < workers ? (uint32_t)enough : workers;
}

static MxPlan plan_of(const Mx4Product &p, uint32_t sms, bool quantises)
{
    MxPlan plan = {};
    const bool by_expert = p.offsets != nullptr;
    const uint32_t typical = by_expert ? (p.m + p.experts - 1u) / p.experts : p.m;
    auto tok_tiles = [&] {
        return by_expert ? (unsigned long long)p.m / plan.ntok + (p.experts < p.m ? p.experts : p.m)
                         : ((unsigned long long)p.m + plan.ntok - 1u) / plan.ntok;
    };
    // Many rows of x, more tiles than blocks (18432 x 4096 by 256 rows: a tile a block 14.2 us, pairs 20.4) and tiles for every pair:
    // 256 rows of w by up to 192 of x.  What two blocks multiply is a multiple of 32 rows of x: not where it would be a sixth more than
    // there are (28672 x 4096 by 208 rows 26.4 us, single blocks 25.0).
    const uint32_t row_tiles = row_tiles_of(p.n, kMxOne);
    const bool one_each = !by_expert && (unsigned long long)((p.m + kMxMaxTok - 1u) / kMxMaxTok) * row_tiles <= sms;
    if (!quantises && !one_each && typical >= kMxPairFrom) {
        const uint32_t parts = (typical + kMxPairTok - 1u) / kMxPairTok;
        const uint32_t ntok = up_to((typical + parts - 1u) / parts, 32u);
        if ((unsigned long long)parts * row_tiles_of(p.n, kMxPair) * p.experts >= sms / 2u
            && (by_expert || parts == 1u || (parts * ntok - typical) * 6u <= typical)) {
            plan.form = kMxPair;
            plan.ntok = ntok;
            deal(plan, tok_tiles() * row_tiles_of(p.n, kMxPair), steps_of(p.k, kMxPair), sms / 2u);
            plan.grid *= 2u;
            return plan;
        }
    }
    // Rows of x per tile: equal parts of at most 256, more of them while there is an SM for each tile, or few enough for clusters.  By
    // expert half as many again as one has on average, so that most need one tile (128 experts of 1536 x 2048 with 32 rows each, by 48
    // rows 41.8 us, by 32 44.9, by 64 43.5; with 16 rows each, by 32 38.9, by 16 41.0).
    const uint32_t steps = steps_of(p.k, kMxOne);
    if (by_expert && typical <= kMxTwoTok) {
        const uint32_t ample = typical + typical / 2u;
        plan.ntok = up_to(ample < kMxTwoTok ? ample : kMxTwoTok, 16u);
    } else {
        uint32_t parts = (typical + kMxMaxTok - 1u) / kMxMaxTok;
        if (!by_expert) {
            const uint32_t most = (p.m + kMxClusterTok - 1u) / kMxClusterTok;
            const uint32_t room = sms / row_tiles < most ? sms / row_tiles : most;
            parts = room > parts ? room : parts;
            for (uint32_t tok = kMxTwoClusterTok; tok <= kMxClusterTok; tok *= 2u) {
                const uint32_t narrow = (p.m + tok - 1u) / tok;
                if ((unsigned long long)narrow * row_tiles <= kMxClustersOf2) {
                    parts = narrow;
                    break;
                }
            }
        }
        plan.ntok = up_to((typical + parts - 1u) / parts, 16u);
    }
    const unsigned long long tiles = tok_tiles() * row_tiles;
    // Few tiles: clusters that share one, if the host knows how many there are, else a tile a block (fewer, if the device finds fewer).
    if (!by_expert) {
        const bool known = p.m_dev == nullptr || tok_tiles() == 1ull;
        for (uint32_t c = 8u; c >= 2u && known && plan.ntok <= kMxClusterTok; c >>= 1) {
            const uint32_t least = c != 2u ? c * kMxClusterSteps
                : plan.ntok <= kMxTwoClusterTok ? kMxClusterSteps2 : kMxClusterSteps2Wide;
            const uint32_t runs = c == 8u ? kMxClustersOf8 : c == 4u ? kMxClustersOf4 : kMxClustersOf2;
            if (tiles <= (plan.ntok <= kMxTwoClusterTok ? 2u * runs : runs) && steps >= least) {
                plan.form = plan.ntok <= kMxTwoClusterTok ? kMxTwo : kMxOne;
                plan.cluster = c;
                plan.grid = (uint32_t)tiles * c;
                return plan;
            }
        }
        if (tiles <= sms || (!quantises && tiles <= 2u * sms && plan.ntok <= kMxTwoTok)) {
            plan.form = tiles <= sms ? kMxOne : kMxTwo;
            plan.grid = (uint32_t)tiles;
            return plan;
        }
    }
    plan.form = plan.ntok <= kMxTwoTok ? kMxTwo : kMxOne;
    deal(plan, tiles, steps, plan.form == kMxTwo ? 2u * sms : sms);
    return plan;
}

// The plan of mx4_linear for few rows: the stages of x that a block needs have to fit beside a ring of weights.
static MxPlan linear_plan(const Mx4Product &p, uint32_t sms)
{
    MxPlan plan = plan_of(p, sms, true);
    if (p.m > kMxFusedRows) {
        return plan;
    }
    const uint32_t steps = steps_of(p.k, plan.form);
    const unsigned long long units = (unsigned long long)row_tiles_of(p.n, plan.form) * steps;
    const uint32_t bytes = plan.ntok * kMxStageBytes + 2u * kMxScaleBlock;
    auto slots = [&] {
        const uint32_t run = plan.cluster != 0u ? (steps + plan.cluster - 1u) / plan.cluster
                                                : (uint32_t)((units + plan.grid - 1u) / plan.grid);
        return run < steps ? run : steps;
    };
    const uint32_t all = slots();
    if (all <= kMxMaxSlots && p.m * all <= kMxFusedWork && all * bytes <= mx_rings(plan.form) * 2u / 5u) {
        plan.slots = all;
    }
    return plan;
}

bool mx4_linear_quantizes(uint32_t n, uint32_t k, uint32_t m, unsigned int sm_count)
{
    Mx4Product p = {};
    p.experts = 1u;
    p.n = n;
    p.k = k;
    p.m = m;
    return linear_plan(p, sm_count).slots != 0u;
}

cudaError_t launch_mx4_product(cudaStream_t stream, const UmmaScratch &scratch, unsigned int sm_count, unsigned int set,
                               const Mx4Product &p)
{
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
    args.status = scratch.status;
    args.partial = scratch.partial + (unsigned long long)(set & 1u) * scratch.blocks * scratch.tile_floats;
    args.flags = scratch.flags + (unsigned long long)(set & 1u) * scratch.blocks * kFlagWords;
    args.tile_floats = scratch.tile_floats;
    const uint32_t size = p.y_dtype == 0 ? 4u : 2u;
    args.wide = (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0u && (args.ldy * size) % 16u == 0u;
    const uint32_t blocks = sm_count < scratch.blocks ? sm_count : scratch.blocks;
    const MxPlan plan = p.x != nullptr ? linear_plan(p, blocks) : plan_of(p, blocks, false);
    const bool pair = plan.form == kMxPair;
    const MxForm form = plan.form;
    args.ntok = plan.ntok;
    args.slots = plan.slots;
    args.cluster = plan.cluster;
    if (p.x != nullptr) {
        args.x = p.x;
        args.x_type = (uint32_t)p.x_dtype;
        args.ldx = p.ldx;
        args.x_aligned = (reinterpret_cast<uintptr_t>(p.x) & 15u) == 0u && (p.ldx * (p.x_dtype == 0 ? 4u : 2u)) % 16u == 0u;
    }
    const uint32_t x_blocks = mx_scale_blocks(args.ntok);
    const uint32_t x_rows = pair ? args.ntok / 2u : args.ntok;
    const uint32_t x_bytes = mx_parts(form) * (x_rows * kMxStageBytes + 2u * x_blocks * kMxScaleBlock);
    args.stage_bytes = mx_parts(form) * (kMxRows + (args.slots != 0u ? 0u : x_rows)) * kMxStageBytes;
    args.scale_bytes = mx_parts(form) * 2u * (1u + (args.slots != 0u ? 0u : x_blocks)) * kMxScaleBlock;
    const uint32_t tile_rows = p.m < args.ntok ? p.m : args.ntok;
    args.share = plan.cluster != 0u ? up_to((tile_rows + plan.cluster - 1u) / plan.cluster, 4u) : 0u;
    const uint32_t exchange = args.cluster * args.share * kMxRows * 4u;
    const uint32_t room = mx_rings(form) - exchange - args.slots * x_bytes;
    const uint32_t fit = room / (args.stage_bytes + args.scale_bytes);
    args.stages = fit < kMxMaxStages ? fit : kMxMaxStages;
    const uint32_t scales = pair ? (room - args.stages * args.stage_bytes) / args.scale_bytes : args.stages;
    args.scale_slots = scales < kMxMaxScales ? scales : kMxMaxScales;
    // Tensor memory: two accumulators where they fit beside scales, and those of as many stages as then fit, two at least (a
    // single block copies a stage's scales without asking for the place: it has one for each).
    const uint32_t stage_columns = mx_parts(form) * 8u * (1u + x_blocks);
    const uint32_t least = pair ? 2u * stage_columns : args.stages * stage_columns;
    args.accumulators = 2u * args.ntok + least <= 512u ? 2u : 1u;
    const uint32_t places = (512u - args.accumulators * args.ntok) / stage_columns;
    args.scale_places = places < args.stages ? places : args.stages;
    const uint32_t columns = args.accumulators * args.ntok + args.scale_places * stage_columns;
    args.tmem_columns = 32u;
    while (args.tmem_columns < columns) {
        args.tmem_columns *= 2u;
    }
    CUtensorMap map_w, map_x = {};
    if (!map_codes(encode, &map_w, p.w_codes, args.w_rows, p.k, kMxRows)
        || (args.slots == 0u && !map_codes(encode, &map_x, p.x_codes, p.m, p.k, x_rows))) {
        return cudaErrorInvalidValue;
    }
    switch (p.y_dtype) {
    case 0:
        return launch_typed<float>(stream, plan.grid, form, map_w, map_x, args, p.overlap);
    case 1:
        return launch_typed<__half>(stream, plan.grid, form, map_w, map_x, args, p.overlap);
    default:
        return launch_typed<__nv_bfloat16>(stream, plan.grid, form, map_w, map_x, args, p.overlap);
    }
}

} // namespace q8
