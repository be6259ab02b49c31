// The pairs of a routed layer in the order of their experts: a stable counting sort, so that a pair's place, and with it the
// tile it lands in, is a function of the selections alone.
#include "mx4.h"
#include "q8_common.cuh"
#include "q8_launch.h"

namespace q8 {

constexpr uint32_t kOrderThreads = 1024;
constexpr uint32_t kOrderWarps = kOrderThreads / 32u;

// One block.  Each warp takes a run of the pairs: it counts them by expert; running totals over the warps and over the
// experts give each warp its first place per expert; then it walks its run again and places the pairs, lanes in order
// within a step (lanes with the same expert find each other with a match).
__global__ void __launch_bounds__(kOrderThreads)
mx4_order_kernel(const uint32_t *ids, uint32_t tokens_max, const uint32_t *tokens_dev, uint32_t used, uint32_t experts,
                 uint32_t *__restrict__ order, uint32_t *__restrict__ token_of, uint32_t *__restrict__ offsets)
{
    __shared__ uint32_t place[kOrderWarps][kMx4MaxExperts];
    __shared__ uint32_t warp_total[kOrderWarps];
    __shared__ uint32_t placed;
    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31u;
    for (uint32_t e = lane; e < kMx4MaxExperts; e += 32u) {
        place[warp][e] = 0u;
    }
    __syncwarp();
    grid_dependency_wait();
    grid_launch_dependents();
    uint32_t tokens = tokens_max;
    if (tokens_dev != nullptr) {
        const uint32_t live = *tokens_dev;
        tokens = live < tokens_max ? live : tokens_max;
    }
    const uint32_t all = tokens_max * used;
    const uint32_t pairs = tokens * used;
    const uint32_t per_warp = ((pairs + kOrderWarps - 1u) / kOrderWarps + 31u) / 32u * 32u;
    const uint32_t begin = warp * per_warp < pairs ? warp * per_warp : pairs;
    const uint32_t end = begin + per_warp < pairs ? begin + per_warp : pairs;
    for (uint32_t p = begin + lane; p < end; p += 32u) {
        const uint32_t e = ids[p];
        if (e < experts) {
            atomicAdd(&place[warp][e], 1u);
        }
    }
    __syncthreads();
    // thread e: expert e
    uint32_t mine = 0u;
    if (threadIdx.x < kMx4MaxExperts) {
        for (uint32_t w = 0; w < kOrderWarps; ++w) {
            const uint32_t here = place[w][threadIdx.x];
            place[w][threadIdx.x] = mine;
            mine += here;
        }
    }
    uint32_t through = mine;
#pragma unroll
    for (uint32_t step = 1u; step < 32u; step <<= 1) {
        const uint32_t below = __shfl_up_sync(0xFFFFFFFFu, through, step);
        if (lane >= step) {
            through += below;
        }
    }
    if (lane == 31u) {
        warp_total[warp] = through;
    }
    __syncthreads();
    if (threadIdx.x < kMx4MaxExperts) {
        for (uint32_t w = 0; w < warp; ++w) {
            through += warp_total[w];
        }
        for (uint32_t w = 0; w < kOrderWarps; ++w) {
            place[w][threadIdx.x] += through - mine;
        }
        if (threadIdx.x < experts) {
            offsets[threadIdx.x + 1u] = through;
            if (threadIdx.x == experts - 1u) {
                placed = through;
            }
        }
        if (threadIdx.x == 0u) {
            offsets[0] = 0u;
        }
    }
    __syncthreads();
    for (uint32_t first = begin; first < end; first += 32u) {
        const uint32_t p = first + lane;
        uint32_t e = p < end ? ids[p] : 0xFFFFFFFFu;
        e = e < experts ? e : 0xFFFFFFFFu;
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
        const uint32_t below = (uint32_t)__popc(same & ((1u << lane) - 1u));
        const uint32_t at = e != 0xFFFFFFFFu ? place[warp][e] + below : 0u;
        __syncwarp();
        if (e != 0xFFFFFFFFu) {
            order[at] = p;
            if (token_of != nullptr) {
                token_of[at] = p / used;
            }
            if (below == 0u) {
                place[warp][e] = at + (uint32_t)__popc(same);
            }
        }
        __syncwarp();
    }
    for (uint32_t at = placed + threadIdx.x; at < all; at += kOrderThreads) {
        order[at] = 0xFFFFFFFFu;
        if (token_of != nullptr) {
            token_of[at] = 0xFFFFFFFFu;
        }
    }
}

cudaError_t launch_mx4_order(cudaStream_t stream, bool overlap, const uint32_t *ids, uint32_t tokens,
                             const uint32_t *tokens_dev, uint32_t used, uint32_t experts, uint32_t *order, uint32_t *token_of,
                             uint32_t *offsets)
{
    return launch_kernel_early(overlap, mx4_order_kernel, dim3(1), kOrderThreads, 0, stream, ids, tokens, tokens_dev, used,
                               experts, order, token_of, offsets);
}

} // namespace q8
