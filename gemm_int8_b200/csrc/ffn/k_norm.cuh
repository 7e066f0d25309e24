// Root-mean-square norm of x (+ residual) in 8 bits, and the sum:
//   h = x + residual (fp32),  total = h rounded to the residual's type,  r = (mean(h^2) + eps)^-1/2,  v = (h r) weight,
//   q, s = 8-bit values and scales of v (out8.cuh), a scale per 128 columns or one per row.
// The norm is of the sum in fp32, not of the total that is stored: one rounding less on the way to q.
//
// One pass: a row is read once, stays in registers (8 LOADS values a thread) while its squares are summed up across its warps (and with per-row scales its largest
// magnitude found), and is written once.  Bound: HBM: 16384 x 8192 bf16 with a residual 141 - 150 us by machine, 6.3 - 6.7 TB/s (a copy: 6.55); 8191 x 4096 bf16 onto an
// fp32 residual 60 us, 6.1 TB/s; without a residual, 3 bytes an element, the latency of a row's steps: 16384 x 4096 50 us, 4 TB/s.  Persistent CTAs that request the next row
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

GI8_DEVICE float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The sum over a row, in an order that is the same in the forms of two and four loads, so that a row's result does not depend on its batch (the form of eight is
// the only one for its widths).  A thread of four loads adds up two parts, its loads 0 and 2, and 1 and 3; of the form of two loads, which has twice the threads, the
// first half of the threads have the first part and are sent the second by the others.  Then over the lanes of a warp, and over the warps.
GI8_DEVICE float row_sum(const float (&part)[2], float*, float* slots, int row_warps)
{
    const int lane = threadIdx.x & 31;
    float v = warp_sum(part[0] + part[1]);
    if (row_warps == 1) return v;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < row_warps ? slots[lane] : 0.0f);
}

GI8_DEVICE float row_sum(const float (&part)[1], float* sent, float* slots, int row_warps)
{
    const int lane = threadIdx.x & 31, warps = row_warps / 2, t = threadIdx.x - warps * 32;
    if (t >= 0) sent[t] = part[0];
    __syncthreads();
    if (t < 0) {  // (a whole warp)
        const float v = warp_sum(part[0] + sent[threadIdx.x]);
        if (lane == 0) slots[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    return warp_sum(lane < warps ? slots[lane] : 0.0f);
}

GI8_DEVICE float row_max(float v, float* slots, int row_warps)
{
    v = warp_max_nan(v);
    if (row_warps == 1) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_max_nan(lane < row_warps ? slots[lane] : 0.0f);
}

// (At most 64 registers where a thread has 32 values, so that two CTAs of 512 threads fit on an SM; most e4m3 forms spill 4 to 12 bytes for it.  With 70 and 76: 16384 x 16384 with a
// residual 371 us for 281, without one 297 for 202, x 8192 without one 108 for 96, x 4096 55 for 50; narrower rows with a residual within 2 %, either way.)
template <typename TX, typename TR, typename TW, Out8 OUT, bool BLOCK, int LOADS>
__global__ void __launch_bounds__(kNormThreads, LOADS == 4 ? 2 : 0) rms_norm_quantize_kernel(const NormParams p)
{
    quant_dependency();
    constexpr bool RESIDUAL = !std::is_same<TR, void>::value;
    using TS = typename std::conditional<RESIDUAL, TR, TX>::type;
    constexpr int PARTS = LOADS == 2 ? 1 : 2;
    __shared__ float slots[3][32], sent[PARTS == 1 ? kNormThreads / 2 : 1];
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
    uint64_t sum2[PARTS];     // of squares
    auto add_squares = [&](int u, const uint64_t (&h)[4]) {
        uint64_t& sum = sum2[u % PARTS];
        sum = u < PARTS ? mul2(h[0], h[0]) : fma2(h[0], h[0], sum);
#pragma unroll
        for (int i = 1; i < 4; ++i) sum = fma2(h[i], h[i], sum);
    };
    auto row_total = [&](float* at) {
        float part[PARTS], lo, hi;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            f32x2_split(sum2[i], lo, hi);
            part[i] = lo + hi;
        }
        return row_sum(part, sent, at, p.row_warps);
    };
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
        add_squares(u, h);
    }
    if constexpr (RESIDUAL) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int col = (u * row_threads + t) * 8;
            if (live && col < p.H) store8(static_cast<TS*>(p.total) + base + col, kept[u]);
        }
    }
    const float sum = row_total(slots[0]);
    float r = rsqrtf(fmaf(sum, p.inv_h, p.eps));
    // Squares that fp32 cannot hold (values from about 1e17 on): once more from values 2^80 times smaller, next to which eps is nothing.
    // (All threads that meet at the reduction's barrier hold the same sum.)
    if (sum > 1e37f) {
        const uint64_t down = f32x2(0x1p-80f, 0x1p-80f);
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const uint64_t h[4] = {mul2(kept[u][0], down), mul2(kept[u][1], down), mul2(kept[u][2], down), mul2(kept[u][3], down)};
            add_squares(u, h);
        }
        r = rsqrtf(row_total(slots[1]) * p.inv_h) * 0x1p-80f;
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
        qs[0] = make_out_scale<OUT>(row_max(top, slots[2], p.row_warps));
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
