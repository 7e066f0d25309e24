// Root-mean-square norm of x (+ residual) in 8 bits, and the sum:
//   h = x + residual (fp32),  total = h rounded to the residual's type,  r = (mean(h^2) + eps)^-1/2,  v = (h r) weight,
//   q, s = 8-bit values and scales of v (out8.cuh), a scale per 128 columns or one per row.
// The norm is of the sum in fp32, not of the total that is stored: one rounding less on the way to q.
//
// One pass: a row is read once, stays in registers (8 LOADS values a thread) while its squares are summed up across its warps (and with per-row scales its largest
// magnitude found), and is written once.  Bound: HBM: 16384 x 8192 bf16 with a residual 141 - 150 us by machine, 6.3 - 6.7 TB/s, the copy rate; 8191 x 4096 bf16 onto an fp32 residual
// 60 us, 6.1 TB/s; without a residual, 3 bytes an element, the latency of a row's steps: 16384 x 4096 50 us, 4 TB/s.  Persistent CTAs that request the next row
// before they work on this one were no faster (150, 65, 58 us): registers for two rows halve the rows on an SM.
#pragma once

#include <type_traits>

#include "out8.cuh"

namespace gi8 {

constexpr int kNormThreads = 512;  // of a CTA, at most

struct NormParams {
    const void* x;         // [M, H]
    const void* residual;  // [M, H]
    const void* weight;    // [H]
    void* total;           // [M, H]; may be the residual or x itself: a thread writes what it alone has read
    uint8_t* q;            // [M, H]
    float* s;              // [M, KB] or [M]
    int64_t M;
    int H, KB;
    int row_warps;         // warps of a row: all of the CTA's, or one
    float eps, inv_h;
};

// The sum of the row's values over its warps' lanes, in a fixed order (MAX: their maximum).
template <bool MAX>
GI8_DEVICE float row_reduce(float v, float* slots, int row_warps)
{
    auto warp_all = [](float x) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float w = __shfl_xor_sync(0xffffffffu, x, o);
            x = MAX ? max_nan(x, w) : x + w;
        }
        return x;
    };
    v = warp_all(v);
    if (row_warps == 1) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_all(lane < row_warps ? slots[lane] : 0.0f);
}

// (At most 64 registers where a thread has 32 values, so that two CTAs of 512 threads fit on an SM; e4m3 spills 4 to 12 bytes for it.  With 70 and 76: 16384 x 16384 with a
// residual 371 us for 281, without one 297 for 202, x 8192 without one 108 for 96, x 4096 55 for 50; narrower rows with a residual within 2 %, either way.)
template <typename TX, typename TR, typename TW, Out8 OUT, bool BLOCK, int LOADS>
__global__ void __launch_bounds__(kNormThreads, LOADS == 4 ? 2 : 0) rms_norm_quantize_kernel(const NormParams p)
{
    quant_dependency();
    constexpr bool RESIDUAL = !std::is_same<TR, void>::value;
    using TS = typename std::conditional<RESIDUAL, TR, TX>::type;
    __shared__ float slots[3][32];
    const int row_threads = p.row_warps * 32;
    const int t = p.row_warps == 1 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = p.row_warps == 1 ? static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const bool live = row < p.M;
    const int64_t base = row * p.H;

    Raw8<TX> raw[LOADS];
    [[maybe_unused]] Raw8<TS> raw_r[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        const int col = (u * row_threads + t) * 8;
        const bool in = live && col < p.H;
        raw[u] = in ? load8(static_cast<const TX*>(p.x) + base + col) : zero8<TX>();
        if constexpr (RESIDUAL) raw_r[u] = in ? load8(static_cast<const TS*>(p.residual) + base + col) : zero8<TS>();
    }
    // A bf16 weight is requested with the row, not behind the reduction (the registers of an fp32 one would cost resident CTAs).
    constexpr bool EARLY = sizeof(TW) == 2 && !RESIDUAL;
    [[maybe_unused]] Raw8<TW> raw_w[LOADS];
    auto load_weight = [&](int u) {
        const int col = (u * row_threads + t) * 8;
        return col < p.H ? load8(static_cast<const TW*>(p.weight) + col) : zero8<TW>();
    };
    if constexpr (EARLY) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) raw_w[u] = load_weight(u);
    }
    uint64_t kept[LOADS][4];  // the sums, then the values
    uint64_t sum2 = 0ull;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        uint64_t (&h)[4] = kept[u];
        unpack8<TX>(raw[u], h);
        if constexpr (RESIDUAL) {
            uint64_t w[4];
            unpack8<TS>(raw_r[u], w);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = add2(h[i], w[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum2 = fma2(h[i], h[i], sum2);
    }
    if constexpr (RESIDUAL) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int col = (u * row_threads + t) * 8;
            if (live && col < p.H) store8(static_cast<TS*>(p.total) + base + col, kept[u]);
        }
    }
    float lo, hi;
    f32x2_split(sum2, lo, hi);
    float sum = row_reduce<false>(lo + hi, slots[0], p.row_warps);
    float r = rsqrtf(fmaf(sum, p.inv_h, p.eps));
    // Squares that fp32 cannot hold (values from about 1e17 on): once more from values 2^80 times smaller, next to which eps is nothing.
    // (All threads that meet at the reduction's barrier hold the same sum.)
    if (sum > 1e37f) {
        const uint64_t down = f32x2(0x1p-80f, 0x1p-80f);
        sum2 = 0ull;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint64_t h = mul2(kept[u][i], down);
                sum2 = fma2(h, h, sum2);
            }
        }
        f32x2_split(sum2, lo, hi);
        r = rsqrtf(row_reduce<false>(lo + hi, slots[2], p.row_warps) * p.inv_h) * 0x1p-80f;
    }
    const uint64_t r2 = f32x2(r, r);
    float m[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        uint64_t w[4];
        if constexpr (EARLY) unpack8<TW>(raw_w[u], w);
        else unpack8<TW>(load_weight(u), w);
#pragma unroll
        for (int i = 0; i < 4; ++i) kept[u][i] = mul2(mul2(kept[u][i], r2), w[i]);
        m[u] = amax8_nan(kept[u]);
    }
    QuantScale qs[BLOCK ? LOADS : 1];
    if constexpr (BLOCK) {
        block_scales<OUT, LOADS>(m, qs);
    } else {
        float top = m[0];
#pragma unroll
        for (int u = 1; u < LOADS; ++u) top = max_nan(top, m[u]);
        qs[0] = make_out_scale<OUT>(row_reduce<true>(top, slots[1], p.row_warps));
        if (live && t == 0) p.s[row] = qs[0].s;
    }
    out8_store<OUT>(kept, qs, [&](int u, uint2 w) {
        const int col = (u * row_threads + t) * 8;
        if (live && col < p.H) {
            if (BLOCK && (t & 15) == 0) p.s[row * p.KB + (col >> 7)] = qs[BLOCK ? u : 0].s;
            *reinterpret_cast<uint2*>(p.q + base + col) = w;
        }
    });
}

}  // namespace gi8
