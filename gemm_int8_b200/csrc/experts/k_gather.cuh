// Token rows in the order of their experts: dst[p] = x[slots[p] / top_k] for p < offsets[E].  In front of the products of many rows, whose
// tiles then are one TMA box each: gathering 128 rows in the product itself, four per TMA instruction, takes three times as long as their
// MMAs (32768 gathered rows, 4096 x 4096: 2010 us; with this pass in front of it about 30 us more than rows that lie in order).
// Bound by HBM: every row is read (tokens from L2, which have top_k readers) and written once.
#pragma once

#include "../ptx.cuh"

namespace gi8 {

constexpr int kGatherThreads = 256;

__global__ void __launch_bounds__(kGatherThreads)
gather_rows_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ slots, const int32_t* __restrict__ last_offset, uint4* __restrict__ dst,
                   int64_t rows, int tokens, int top_k, int chunks)
{
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t kept = min(static_cast<int64_t>(__ldg(last_offset)), rows);
    for (int64_t p = static_cast<int64_t>(blockIdx.x) * (kGatherThreads / 32) + (threadIdx.x >> 5); p < kept; p += static_cast<int64_t>(gridDim.x) * (kGatherThreads / 32)) {
        const int token = min(max(__ldg(slots + p), 0) / top_k, tokens - 1);
        const uint4* from = x + static_cast<int64_t>(token) * chunks;
        uint4* to = dst + p * chunks;
        for (int c0 = lane; c0 < chunks; c0 += 32 * 8) {
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + 32 * i < chunks) v[i] = __ldg(from + c0 + 32 * i);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c0 + 32 * i < chunks) to[c0 + 32 * i] = v[i];
        }
    }
}

}  // namespace gi8
