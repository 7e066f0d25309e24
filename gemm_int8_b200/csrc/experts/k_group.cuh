// Groups the (token, choice) pairs of a routed batch by expert: a stable counting sort of S = T k expert ids.
//   offsets [E + 1]  rows [offsets[e], offsets[e + 1]) belong to expert first + e
//   slots   [S]      slots[p] = t k + j of the pair in row p, ascending within an expert; -1 behind offsets[E]
//   places  [S]      the inverse: the row of pair t k + j, or -1 for a pair whose expert is not one of the E here
//
// Every warp owns a run of consecutive pairs, which it reads once into registers, and counts them per expert in a histogram row of its own
// (the lanes with equal ids find one another, and one of them adds their number), which also gives each pair its rank in the run; the
// warps' rows are summed up per expert, and a pair's row is its rank plus what lies in front of its warp.  A CTA's pairs are put in order in
// shared memory before they leave, as runs of an expert instead of one 32-byte sector for each.  No atomics: the result does not depend
// on timing.  Up to 8192 pairs one CTA does it all; more are counted by one launch and placed by a second one, which adds up the counts of the
// CTAs in front of its own.  Bound by latencies and launches: 131072 pairs of 256 experts 8.2 us, of which two empty launches take
// 3.6 (in one launch of a cluster of eight CTAs, which exchange their counts through distributed shared memory, 20.9: eight SMs are too few).
#pragma once

#include "../ptx.cuh"

namespace gi8 {

constexpr int kGroupMaxExperts = 1024;

struct GroupParams {
    const int32_t* experts;  // [S]
    int32_t* offsets;        // [E + 1]
    int32_t* slots;          // [S]
    int32_t* places;         // [S]
    int32_t* counts;         // [CTAs][E], between the two launches
    int S, E, first;
    int per_warp;            // pairs of a warp's run, at most 32 LOADS
    int bits;                // of an id, 0 .. E
};

enum GroupStep : int { GROUP_ALL, GROUP_COUNT, GROUP_PLACE };

// The lanes that have the same id, of `bits` bits: a ballot per bit (match.any takes about twice as long where most ids differ).
GI8_DEVICE uint32_t same_id(int id, int bits)
{
    uint32_t same = 0xffffffffu;
#pragma unroll
    for (int b = 0; b < 11; ++b) {
        if (b >= bits) break;
        const bool one = (id >> b) & 1;
        const uint32_t ones = __ballot_sync(0xffffffffu, one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// Shared memory, in words: per warp and expert [WARPS][E], totals [E], first [E], shift [E], the CTA's pairs [WARPS * 32 * LOADS]; the third
// and fourth are [parts][E] and [parts][E] while the other CTAs' counts are added up.
template <int WARPS, int LOADS, GroupStep STEP>
__global__ void __launch_bounds__(WARPS * 32)
group_by_expert_kernel(const GroupParams p)
{
    extern __shared__ int32_t group_smem[];
    __shared__ int32_t warp_sums[2][32];
    __shared__ int32_t carry_slot[2];
    constexpr int kThreads = WARPS * 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int32_t* by_warp = group_smem;
    int32_t* totals = by_warp + WARPS * p.E;
    int32_t* own_first = totals + p.E;  // where an expert's pairs begin among this CTA's,
    int32_t* shift = own_first + p.E;   // and how much further on among all
    int32_t* sorted = shift + p.E;
    for (int i = tid; i < WARPS * p.E; i += kThreads) by_warp[i] = 0;
    if (tid < 2) carry_slot[tid] = 0;
    pdl_wait();
    if (tid == 0) pdl_launch_dependents();

    const int64_t cta_begin = static_cast<int64_t>(blockIdx.x) * WARPS * p.per_warp;
    const int64_t begin = cta_begin + static_cast<int64_t>(warp) * p.per_warp;
    const int run = static_cast<int>(min(static_cast<int64_t>(p.per_warp), max(static_cast<int64_t>(0), p.S - begin)));
    int32_t* mine = by_warp + warp * p.E;
    int id[LOADS], rank[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int i = j * 32 + lane;
        const int64_t e = i < run ? static_cast<int64_t>(__ldg(p.experts + begin + i)) - p.first : -1;
        id[j] = e >= 0 && e < p.E ? static_cast<int>(e) : p.E;  // E: not one of ours
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        if (j * 32 < run) {
            const uint32_t same = same_id(id[j], p.bits);
            const int before = id[j] < p.E ? mine[id[j]] : 0;
            rank[j] = before + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (id[j] < p.E && lane == __ffs(same) - 1) mine[id[j]] = before + __popc(same);
            __syncwarp();
        }
    }
    __syncthreads();
    // per expert: exclusive sums over the warps, the CTA's total
    for (int e = tid; e < p.E; e += kThreads) {
        int32_t n[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) n[w] = by_warp[w * p.E + e];
        int32_t sum = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            by_warp[w * p.E + e] = sum;
            sum += n[w];
        }
        totals[e] = sum;
        if constexpr (STEP == GROUP_COUNT) p.counts[static_cast<int64_t>(blockIdx.x) * p.E + e] = sum;
    }
    if constexpr (STEP == GROUP_COUNT) return;

    // all CTAs' totals, and those of the CTAs in front of this one: rows of counts dealt to as many threads per expert as there are
    int32_t *sum_all = own_first, *sum_before = own_first;
    int parts = 1;
    if constexpr (STEP == GROUP_PLACE) {
        parts = max(1, min(kThreads / p.E, LOADS * kThreads / (2 * p.E)));  // (they lie over the CTA's pairs)
        sum_all = sorted, sum_before = sorted + parts * p.E;
        for (int i = tid; i < parts * p.E; i += kThreads) {
            const int part = i / p.E, e = i - part * p.E;
            int32_t all = 0, before = 0;
#pragma unroll 16
            for (int c = part; c < static_cast<int>(gridDim.x); c += parts) {
                const int32_t n = __ldcg(p.counts + static_cast<int64_t>(c) * p.E + e);
                all += n;
                before += c < static_cast<int>(blockIdx.x) ? n : 0;
            }
            sum_all[i] = all, sum_before[i] = before;
        }
    }
    __syncthreads();
    // exclusive sums over the experts, of all CTAs' totals and of this CTA's
    for (int base = 0; base < p.E; base += kThreads) {
        const int e = base + tid;
        int32_t all = 0, before = 0, own = 0;
        if (e < p.E) {
            own = all = totals[e];
            if constexpr (STEP == GROUP_PLACE) {
                all = 0;
                for (int q = 0; q < parts; ++q) all += sum_all[q * p.E + e], before += sum_before[q * p.E + e];
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
            own_first[e] = start;
            shift[e] = offset + before - start;
            if (blockIdx.x == 0) p.offsets[e] = offset;
        }
        __syncthreads();
        if (tid == kThreads - 1) carry_slot[0] = offset + all, carry_slot[1] = start + own;
        __syncthreads();
    }
    const int32_t kept = carry_slot[0];
    if (blockIdx.x == 0 && tid == 0) p.offsets[p.E] = kept;
    for (int64_t i = kept + static_cast<int64_t>(blockIdx.x) * kThreads + tid; i < p.S; i += static_cast<int64_t>(gridDim.x) * kThreads) p.slots[i] = -1;

    constexpr int kExpertBits = 10;
    static_assert(kGroupMaxExperts <= 1 << kExpertBits && WARPS * 32 * LOADS <= 1 << (31 - kExpertBits), "a pair of the CTA and its expert share a word");
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int i = j * 32 + lane;
        if (i < run) {
            int32_t place = -1;
            if (id[j] < p.E) {
                const int32_t at = own_first[id[j]] + mine[id[j]] + rank[j];
                sorted[at] = static_cast<int32_t>(begin - cta_begin + i) << kExpertBits | id[j];
                place = at + shift[id[j]];
            }
            p.places[begin + i] = place;
        }
    }
    __syncthreads();
    const int held = carry_slot[1];
    for (int i = tid; i < held; i += kThreads) {
        const int32_t v = sorted[i];
        p.slots[i + shift[v & ((1 << kExpertBits) - 1)]] = static_cast<int32_t>(cta_begin) + (v >> kExpertBits);
    }
}

}  // namespace gi8
