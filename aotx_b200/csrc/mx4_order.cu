// The pairs of a routed layer in the order of their experts: a stable counting sort, so that a pair's place, and with it the
// tile it lands in, is a function of the selections alone.
#include "mx4.h"
#include "q8_common.cuh"
#include "q8_launch.h"

namespace q8 {

// Warps: 32, or 8 for few pairs, which are started and synchronised sooner (64 pairs 2.3 us, 512 2.9; with 32 warps, and lanes for warps in
// the running totals, 3.3 and 3.8).
constexpr uint32_t kOrderWarps = 32;
constexpr uint32_t kOrderFewWarps = 8;
constexpr uint32_t kOrderFewPairs = 1024;
constexpr uint32_t kOrderAhead = 4;          // selections per lane whose loads are issued together
constexpr uint32_t kOrderStaged = 32768;     // pairs whose order is made in shared memory, at most

__device__ __forceinline__ void order_load(const uint32_t *ids, uint32_t first, uint32_t end, uint32_t experts, uint32_t lane,
                                           uint32_t (&e)[kOrderAhead])
{
#pragma unroll
    for (uint32_t a = 0; a < kOrderAhead; ++a) {
        const uint32_t p = first + 32u * a + lane;
        e[a] = p < end ? ids[p] : 0xFFFFFFFFu;
    }
#pragma unroll
    for (uint32_t a = 0; a < kOrderAhead; ++a) {
        e[a] = e[a] < experts ? e[a] : 0xFFFFFFFFu;
    }
}

// The lanes with the same expert (what a match gives, which takes 350 cycles of the scheduler; a ballot for each of the number's
// bits 40): e is an expert or 0xFFFFFFFF.
__device__ __forceinline__ uint32_t order_same(uint32_t e, uint32_t bits)
{
    uint32_t same = __ballot_sync(0xFFFFFFFFu, e != 0xFFFFFFFFu);
    same = e != 0xFFFFFFFFu ? same : ~same;
    for (uint32_t b = 0; b < bits; ++b) {
        const bool set = (e >> b & 1u) != 0u;
        const uint32_t with = __ballot_sync(0xFFFFFFFFu, set);
        same &= set ? with : ~with;
    }
    return same;
}

// One block; latency bounds it, and the way of scattered words through one SM: so the order is made in shared memory where it
// fits and goes out in rows (512 tokens with 8 of 128 experts 6.0 us, straight to memory 0.9 more).  Each warp takes a run of
// the pairs and counts them by expert; running totals over the warps, a thread for each expert, and then over the experts give
// each warp its first place per expert; then it places its pairs, lanes in order within a step (lanes with the same expert find each
// other by ballots).
template <uint32_t WARPS>
__global__ void __launch_bounds__(WARPS * 32u)
mx4_order_kernel(const uint32_t *ids, uint32_t tokens_max, const uint32_t *tokens_dev, uint32_t used, uint32_t experts,
                 uint32_t *__restrict__ order, uint32_t *__restrict__ token_of, uint32_t *__restrict__ offsets, bool staged)
{
    extern __shared__ uint32_t sorted[];
    // (an odd distance of rows: a column's words lie in different banks)
    __shared__ uint32_t place[WARPS][kMx4MaxExperts + 1u];
    __shared__ uint32_t sums[kMx4MaxExperts / 32u];
    __shared__ uint32_t begin_of[kMx4MaxExperts];
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
    const uint32_t per_warp = ((pairs + WARPS - 1u) / WARPS + 31u) / 32u * 32u;
    const uint32_t begin = warp * per_warp < pairs ? warp * per_warp : pairs;
    const uint32_t end = begin + per_warp < pairs ? begin + per_warp : pairs;
    const uint32_t bits = 32u - (uint32_t)__clz((int)(experts - 1u));
    uint32_t e[kOrderAhead];
    for (uint32_t first = begin; first < end; first += 32u * kOrderAhead) {
        order_load(ids, first, end, experts, lane, e);
#pragma unroll
        for (uint32_t a = 0; a < kOrderAhead; ++a) {
            if (e[a] != 0xFFFFFFFFu) {
                atomicAdd(&place[warp][e[a]], 1u);
            }
        }
    }
    __syncthreads();
    // a thread an expert: running totals over the warps, then over the experts
    static_assert(WARPS * 32u >= kMx4MaxExperts, "a thread for each expert");
    const uint32_t mine = threadIdx.x;
    uint32_t total = 0u, through = 0u;
    if (mine < kMx4MaxExperts) {
        uint32_t here[WARPS];
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w) {
            here[w] = place[w][mine];
        }
#pragma unroll
        for (uint32_t w = 0; w < WARPS; ++w) {
            place[w][mine] = total;
            total += here[w];
        }
        through = total;
#pragma unroll
        for (uint32_t step = 1u; step < 32u; step <<= 1) {
            const uint32_t below = __shfl_up_sync(0xFFFFFFFFu, through, step);
            through += lane >= step ? below : 0u;
        }
        if (lane == 31u) {
            sums[warp] = through;
        }
    }
    __syncthreads();
    if (mine < kMx4MaxExperts) {
        for (uint32_t w = 0; w < warp; ++w) {
            through += sums[w];
        }
        begin_of[mine] = through - total;
        if (mine <= experts) {
            offsets[mine] = through - total;
        }
        if (mine == kMx4MaxExperts - 1u) {
            placed = through;
            if (experts == kMx4MaxExperts) {
                offsets[kMx4MaxExperts] = through;
            }
        }
    }
    __syncthreads();
    for (uint32_t first = begin; first < end; first += 32u * kOrderAhead) {
        if (per_warp > 32u * kOrderAhead) {
            order_load(ids, first, end, experts, lane, e);       // else they are still there
        }
#pragma unroll
        for (uint32_t a = 0; a < kOrderAhead; ++a) {
            if (first + 32u * a >= end) {
                break;
            }
            const uint32_t p = first + 32u * a + lane;
            const uint32_t same = order_same(e[a], bits);
            const uint32_t below = (uint32_t)__popc(same & ((1u << lane) - 1u));
            const bool in = e[a] != 0xFFFFFFFFu;
            const uint32_t at = in ? place[warp][e[a]] + below : 0u;
            __syncwarp();
            if (in) {
                const uint32_t to = begin_of[e[a]] + at;
                if (staged) {
                    sorted[to] = p;
                } else {
                    order[to] = p;
                    if (token_of != nullptr) {
                        token_of[to] = p / used;
                    }
                }
                if (below == 0u) {
                    place[warp][e[a]] = at + (uint32_t)__popc(same);
                }
            }
            __syncwarp();
        }
    }
    if (staged) {
        __syncthreads();
        for (uint32_t at = threadIdx.x; at < placed; at += WARPS * 32u) {
            const uint32_t p = sorted[at];
            order[at] = p;
            if (token_of != nullptr) {
                token_of[at] = p / used;
            }
        }
    }
    for (uint32_t at = placed + threadIdx.x; at < all; at += WARPS * 32u) {
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
    auto launch = [&](auto kernel, uint32_t warps, bool staged) {
        return launch_kernel_early(overlap, kernel, dim3(1), warps * 32u, staged ? tokens * used * 4u : 0u, stream, ids, tokens, tokens_dev,
                                   used, experts, order, token_of, offsets, staged);
    };
    if (tokens * used <= kOrderFewPairs) {
        return launch(mx4_order_kernel<kOrderFewWarps>, kOrderFewWarps, true);
    }
    static unsigned long long configured = 0ull;
    const cudaError_t err = allow_shared_memory(mx4_order_kernel<kOrderWarps>, kOrderStaged * 4u, &configured);
    if (err != cudaSuccess) {
        return err;
    }
    return launch(mx4_order_kernel<kOrderWarps>, kOrderWarps, tokens * used <= kOrderStaged);
}

} // namespace q8
