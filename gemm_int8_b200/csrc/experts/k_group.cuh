// Groups the (token, choice) pairs of a routed batch by expert: a stable counting sort of S = T k expert ids.
//   offsets [E + 1]  rows [offsets[e], offsets[e + 1]) belong to expert first + e
//   slots   [S]      slots[p] = t k + j of the pair in row p, ascending within an expert; -1 behind offsets[E]
//   places  [S]      the inverse: the row of pair t k + j, or -1 for a pair whose expert is not one of the E here
//
// One cluster of up to eight CTAs does it all in one launch.  Every warp owns a run of consecutive pairs and counts them per expert in
// a histogram row of its own (the lanes with equal ids find one another, and one of them adds their number); the warps' rows are
// summed up per expert, the CTAs' totals are exchanged through distributed shared memory, and a second walk over the ids hands out the
// places.  No atomics: the result does not depend on timing.
#pragma once

#include "../ptx.cuh"

namespace gi8 {

constexpr int kGroupMaxExperts = 1024;

struct GroupParams {
    const int32_t* experts;  // [S]
    int32_t* offsets;        // [E + 1]
    int32_t* slots;          // [S]
    int32_t* places;         // [S]
    int S, E, first;
    int per_warp;            // pairs of a warp's run
};

GI8_DEVICE int32_t ld_dsmem_s32(uint32_t cluster_addr)
{
    int32_t v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}

// Shared memory: counts [WARPS][E], totals [E].
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
group_by_expert_kernel(const GroupParams p, int ctas)
{
    extern __shared__ int32_t group_smem[];
    __shared__ int32_t warp_sums[32];
    __shared__ int32_t carry_slot;
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    constexpr int kThreads = WARPS * 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t* counts = group_smem;
    int32_t* totals = group_smem + WARPS * p.E;
    for (int i = tid; i < WARPS * p.E; i += kThreads) counts[i] = 0;
    if (tid == 0) carry_slot = 0;
    __syncthreads();

    const int64_t begin = (static_cast<int64_t>(blockIdx.x) * WARPS + warp) * p.per_warp;
    const int run = static_cast<int>(min(static_cast<int64_t>(p.per_warp), max(static_cast<int64_t>(0), p.S - begin)));
    int32_t* mine = counts + warp * p.E;
    auto id_at = [&](int i) -> int {  // E: not one of ours
        if (i >= run) return p.E;
        const int64_t e = static_cast<int64_t>(__ldg(p.experts + begin + i)) - p.first;
        return e >= 0 && e < p.E ? static_cast<int>(e) : p.E;
    };
    for (int i = lane; i - lane < run; i += 32) {
        const int e = id_at(i);
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        if (e < p.E && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // per expert: exclusive sums over the warps, the CTA's total
    for (int e = tid; e < p.E; e += kThreads) {
        int32_t sum = 0;
        for (int w = 0; w < WARPS; ++w) {
            const int32_t n = counts[w * p.E + e];
            counts[w * p.E + e] = sum;
            sum += n;
        }
        totals[e] = sum;
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    // exclusive sum over the experts of all CTAs' totals, plus what the CTAs in front of this one have of the same expert
    for (int base = 0; base < p.E; base += kThreads) {
        const int e = base + tid;
        int32_t all = 0, before = 0;
        if (e < p.E) {
            if (ctas > 1) {
                const uint32_t addr = smem_u32(totals + e);
                for (int r = 0; r < ctas; ++r) {
                    const int32_t n = ld_dsmem_s32(map_to_cta(addr, r));
                    if (r < static_cast<int>(blockIdx.x)) before += n;
                    all += n;
                }
            } else {
                all = totals[e];
            }
        }
        int32_t incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_sums[warp] = incl;
        __syncthreads();
        int32_t offset = carry_slot + incl - all;
        for (int w = 0; w < warp; ++w) offset += warp_sums[w];
        if (e < p.E) {
            for (int w = 0; w < WARPS; ++w) counts[w * p.E + e] += offset + before;
            if (blockIdx.x == 0) p.offsets[e] = offset;
        }
        __syncthreads();
        if (tid == kThreads - 1) carry_slot = offset + all;
        __syncthreads();
    }
    const int32_t kept = carry_slot;
    if (blockIdx.x == 0 && tid == 0) p.offsets[p.E] = kept;
    for (int64_t i = kept + static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < p.S; i += static_cast<int64_t>(ctas) * kThreads) p.slots[i] = -1;

    for (int i = lane; i - lane < run; i += 32) {
        const int e = id_at(i);
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const int lead = __ffs(same) - 1;
        int32_t place = -1;
        if (e < p.E) {
            place = mine[e] + __popc(same & ((1u << lane) - 1u));
            p.slots[place] = static_cast<int32_t>(begin + i);
        }
        __syncwarp();
        if (e < p.E && lane == lead) mine[e] += __popc(same);
        __syncwarp();
        if (i < run) p.places[begin + i] = place;
    }
    if (ctas > 1) cluster_sync_all();  // nobody leaves while its totals may still be read
}

}  // namespace gi8
