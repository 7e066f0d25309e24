// Groups the (token, choice) pairs of a routed batch by expert: a stable counting sort of S = T k expert ids.
//   offsets [E + 1]  rows [offsets[e], offsets[e + 1]) belong to expert first + e
//   slots   [S]      slots[p] = t k + j of the pair in row p, ascending within an expert; -1 behind offsets[E]
//   places  [S]      the inverse: the row of pair t k + j, or -1 for a pair whose expert is not one of the E here
//
// One cluster of up to eight CTAs does it all in one launch.  Every warp owns a run of consecutive pairs and counts them per expert in
// a histogram row of its own (the lanes with equal ids find one another, and one of them adds their number), which also gives each pair its
// rank in the run; the warps' rows are summed up per expert, the CTAs' totals are exchanged through distributed shared memory, and a pair's
// row is its rank plus what lies in front of its warp.  No atomics: the result does not depend on timing.
// Bound by latencies and, for large batches, by the eight SMs' stores: a run of at most 32 LOADS pairs is read once, into registers, and
// the CTA's pairs are put in order in shared memory before they leave, as runs of an expert instead of one 32-byte sector for each
// (131072 pairs of 256 experts: 26.2 -> GROUP_US us).  Longer runs are read a second time and leave one by one.
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

// Shared memory, in words: counts [WARPS][E], totals [E], and for runs in registers first [E], shift [E], the CTA's pairs [WARPS * 32 * LOADS].
// LOADS: pairs per lane that are kept in registers; 0: runs of any length.
template <int WARPS, int LOADS>
__global__ void __launch_bounds__(WARPS * 32)
group_by_expert_kernel(const GroupParams p, int ctas)
{
    extern __shared__ int32_t group_smem[];
    __shared__ int32_t warp_sums[2][32];
    __shared__ int32_t carry_slot[2];
    constexpr int kThreads = WARPS * 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t* counts = group_smem;
    int32_t* totals = group_smem + WARPS * p.E;
    int32_t* own_first = totals + p.E;  // where an expert's pairs begin among this CTA's,
    int32_t* shift = own_first + p.E;   // and how much further on among all
    int32_t* sorted = shift + p.E;
    for (int i = tid; i < WARPS * p.E; i += kThreads) counts[i] = 0;
    if (tid < 2) carry_slot[tid] = 0;
    pdl_wait();
    if (tid == 0) pdl_launch_dependents();

    const int64_t cta_begin = static_cast<int64_t>(blockIdx.x) * WARPS * p.per_warp;
    const int64_t begin = cta_begin + static_cast<int64_t>(warp) * p.per_warp;
    const int run = static_cast<int>(min(static_cast<int64_t>(p.per_warp), max(static_cast<int64_t>(0), p.S - begin)));
    int32_t* mine = counts + warp * p.E;
    auto id_at = [&](int i) -> int {  // E: not one of ours
        if (i >= run) return p.E;
        const int64_t e = static_cast<int64_t>(__ldg(p.experts + begin + i)) - p.first;
        return e >= 0 && e < p.E ? static_cast<int>(e) : p.E;
    };
    int id[LOADS > 0 ? LOADS : 1], rank[LOADS > 0 ? LOADS : 1];
    if constexpr (LOADS > 0) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) id[j] = id_at(j * 32 + lane);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            if (j * 32 < run) {
                const uint32_t same = __match_any_sync(0xffffffffu, id[j]);
                const int before = id[j] < p.E ? mine[id[j]] : 0;
                rank[j] = before + __popc(same & ((1u << lane) - 1u));
                __syncwarp();
                if (id[j] < p.E && lane == __ffs(same) - 1) mine[id[j]] = before + __popc(same);
                __syncwarp();
            }
        }
    } else {
        __syncthreads();
        for (int i = lane; i - lane < run; i += 32) {
            const int e = id_at(i);
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            if (e < p.E && lane == __ffs(same) - 1) mine[e] += __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    // per expert: exclusive sums over the warps, the CTA's total
    for (int e = tid; e < p.E; e += kThreads) {
        int32_t n[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) n[w] = counts[w * p.E + e];
        int32_t sum = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            counts[w * p.E + e] = sum;
            sum += n[w];
        }
        totals[e] = sum;
    }
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
    // exclusive sums over the experts, of all CTAs' totals and of this CTA's; what the CTAs in front of this one have of the same expert
    for (int base = 0; base < p.E; base += kThreads) {
        const int e = base + tid;
        int32_t all = 0, before = 0, own = 0;
        if (e < p.E) {
            own = all = totals[e];
            if (ctas > 1) {
                const uint32_t addr = smem_u32(totals + e);
                int32_t n[8];
#pragma unroll
                for (int r = 0; r < 8; ++r) n[r] = r < ctas ? ld_dsmem_s32(map_to_cta(addr, r)) : 0;
                all = 0;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    if (r < static_cast<int>(blockIdx.x)) before += n[r];
                    all += n[r];
                }
            }
        }
        int32_t incl = all, incl_own = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xffffffffu, incl, o), u = __shfl_up_sync(0xffffffffu, incl_own, o);
            if (lane >= o) incl += v, incl_own += u;
        }
        if (lane == 31) warp_sums[0][warp] = incl, warp_sums[1][warp] = incl_own;
        __syncthreads();
        int32_t offset = carry_slot[0] + incl - all, start = carry_slot[1] + incl_own - own;
        for (int w = 0; w < warp; ++w) offset += warp_sums[0][w], start += warp_sums[1][w];
        if (e < p.E) {
            if constexpr (LOADS > 0) {
                own_first[e] = start;
                shift[e] = offset + before - start;
            } else {
                for (int w = 0; w < WARPS; ++w) counts[w * p.E + e] += offset + before;
            }
            if (blockIdx.x == 0) p.offsets[e] = offset;
        }
        __syncthreads();
        if (tid == kThreads - 1) carry_slot[0] = offset + all, carry_slot[1] = start + own;
        __syncthreads();
    }
    if (ctas > 1) cluster_arrive_relaxed();  // the other CTAs' totals have been read
    const int32_t kept = carry_slot[0];
    if (blockIdx.x == 0 && tid == 0) p.offsets[p.E] = kept;
    for (int64_t i = kept + static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < p.S; i += static_cast<int64_t>(ctas) * kThreads) p.slots[i] = -1;

    if constexpr (LOADS > 0) {
        constexpr int kExpertBits = 10;
        static_assert(kGroupMaxExperts <= 1 << kExpertBits && WARPS * 32 * LOADS <= 1 << (31 - kExpertBits), "a pair of the CTA and its expert share a word");
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            if (j * 32 + lane < run) {
                int32_t place = -1;
                if (id[j] < p.E) {
                    const int32_t at = own_first[id[j]] + mine[id[j]] + rank[j];
                    sorted[at] = static_cast<int32_t>(begin - cta_begin + j * 32 + lane) << kExpertBits | id[j];
                    place = at + shift[id[j]];
                }
                p.places[begin + j * 32 + lane] = place;
            }
        }
        __syncthreads();
        const int held = carry_slot[1];
        for (int i = tid; i < held; i += kThreads) {
            const int32_t v = sorted[i];
            p.slots[i + shift[v & ((1 << kExpertBits) - 1)]] = static_cast<int32_t>(cta_begin) + (v >> kExpertBits);
        }
    } else {
        for (int i = lane; i - lane < run; i += 32) {
            const int e = id_at(i);
            const uint32_t same = __match_any_sync(0xffffffffu, e);
            int32_t place = -1;
            if (e < p.E) {
                place = mine[e] + __popc(same & ((1u << lane) - 1u));
                p.slots[place] = static_cast<int32_t>(begin + i);
            }
            __syncwarp();
            if (e < p.E && lane == __ffs(same) - 1) mine[e] += __popc(same);
            __syncwarp();
            if (i < run) p.places[begin + i] = place;
        }
    }
    if (ctas > 1) cluster_wait();  // nobody leaves while its totals may still be read
}

}  // namespace gi8
