// Elementwise activations in 8 bits: the e4m3 quantiser, and SwiGLU behind the product of gate and up rows,
//   v = g / (1 + exp(-g)) u   of the two halves of a row,   in fp32 from fp32 or bf16,
// with a scale per row and 128 columns, or (SwiGLU in int8) one per row.  Every element is read and written once.  Bound: HBM, with instruction issue close behind for
// bf16 input: SwiGLU 4096 x 14336 in e4m3 50 - 55 us by machine, 5.4 - 5.9 TB/s (0.82 - 0.9 of the copy rate; 17 instructions an element issued on 62 % of the cycles), fp32
// 76 - 78 us, 6.8 TB/s; e4m3 quantiser 16384 x 8192 bf16 72 us, 5.7 TB/s, fp32 98 us, 6.9 TB/s; per row 4096 x 14336 60 - 64 us, 4.6 - 4.9 TB/s, fp32 84 - 87 us, 6.1 TB/s
// (a CTA's loads, maximum and stores follow each other; two CTAs of 448 threads share an SM).
#pragma once

#include "out8.cuh"

namespace gi8 {

struct ActParams {
    const void* in;  // [M, K], SwiGLU: [M, 2 K]
    uint8_t* q;      // [M, K]
    float* s;        // [M, KB] or [M]
    int64_t M;
    int K, KB;
};

// g u / (1 + exp(-g)) for a pair, in packed steps but for the exponentials and reciprocals, which the special-function unit takes one by one.
// A product with log2 e that is rounded, by up to |g| / 2^24, would cost the exponential |g| / 2 units in the last place.  So
//   bf16   exp(-g) = 2^t (1 - g d),  t = -g l, l = log2 e to 16 bits, so that t is exact, and d = ln 2 (log2 e - l);  (g d)^2 / 2 is below 1.6 / 2^24
//   fp32   exp(-g) = 2^t (1 - r),    t = -g log2 e rounded, r = g + t ln 2 in one fused step
// and v is good to 14 / 2^24 of itself, next to the half step of 1/254 or 2^-4 that it is rounded by.  (Subnormal exponentials are flushed: next to 1 they are nothing.)
// Without the correction: 4096 x 14336 bf16 47.3 us for 49.8 in e4m3, in int8 level; fp32 level.
// sums: what 1 + exp(-g) adds up to, for act_far.
template <typename T>
GI8_DEVICE uint64_t swiglu2(uint64_t g, uint64_t u, uint64_t& sums)
{
    constexpr float kLog2e = sizeof(T) == 2 ? 1.44268798828125f : 1.44269504f;
    const uint64_t one = f32x2(1.0f, 1.0f), t = mul2(g, f32x2(-kLog2e, -kLog2e));
    float a, b;
    f32x2_split(t, a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    const uint64_t e = f32x2(a, b);
    uint64_t s;  // 1 + exp(-g)
    if constexpr (sizeof(T) == 2) s = fma2(e, fma2(g, f32x2(-4.88849e-6f, -4.88849e-6f), one), one);
    else s = fma2(e, sub2(one, fma2(t, f32x2(0.693147181f, 0.693147181f), g)), one);
    sums = add2(sums, s);
    f32x2_split(s, a, b);
    return mul2(mul2(g, f32x2(approx_reciprocal(a), approx_reciprocal(b))), u);
}

// Gates for which that does not hold: the lowest, whose reciprocals would be subnormal and flushed (from -87.3 on), or whose exponentials overflow while g exp(g) u is
// still a number, infinities and NaN.  (From 1e38 on v is g u either way.)
GI8_DEVICE bool far_gate(float g) { return !(g > -87.0f && g < 1e38f); }

// A lane's sums tell whether it may have met one: exp(87) = 2^125.5, an infinity of either sign (1 - r is rounded), or NaN.
GI8_DEVICE bool act_far(uint64_t sums)
{
    float a, b;
    f32x2_split(sums, a, b);
    return !(fabsf(a + b) <= 0x1p125f);
}

// For them: with y = exp(g/2) for negative g, g u exp(g) / (1 + exp(g)) as (g y) (u y) / (1 + y^2), no part of which underflows before the result does
// (down to -174, from where on y is subnormal and the result below 1e-35 for every u).
GI8_DEVICE float swiglu_far(float g, float u)
{
    const float h = expf(-0.5f * fabsf(g)), y = g < 0.0f ? h : 1.0f;
    return __fdiv_rn(g * y, fmaf(h, h, 1.0f)) * (u * y);
}

template <typename T, bool SWIGLU>
struct ActRaw {
    Raw8<T> a, b;
};

template <typename T>
struct ActRaw<T, false> {
    Raw8<T> a;
};

template <typename T, bool SWIGLU>
GI8_DEVICE ActRaw<T, SWIGLU> act_load(const ActParams& p, int64_t row, int col, bool in)
{
    ActRaw<T, SWIGLU> r;
    const T* at = static_cast<const T*>(p.in) + row * (SWIGLU ? 2 : 1) * static_cast<int64_t>(p.K) + col;
    r.a = in ? load8(at) : zero8<T>();
    if constexpr (SWIGLU) r.b = in ? load8(at + p.K) : zero8<T>();
    return r;
}

template <typename T, bool SWIGLU>
GI8_DEVICE void act_values(const ActRaw<T, SWIGLU>& r, uint64_t (&v)[4], uint64_t& sums)
{
    unpack8<T>(r.a, v);
    if constexpr (SWIGLU) {
        uint64_t w[4];
        unpack8<T>(r.b, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = swiglu2<T>(v[i], w[i], sums);
    }
}

// The same with far gates right.  The others' values are the same to the bit, so that a value depends on nothing beside it.
template <typename T>
GI8_DEVICE void act_values_far(const ActRaw<T, true>& r, uint64_t (&v)[4])
{
    uint64_t g[4], w[4], sums = 0ull;
    act_values<T, true>(r, v, sums);
    if (!act_far(sums)) return;
    unpack8<T>(r.a, g), unpack8<T>(r.b, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float g0, g1, u0, u1, v0, v1;
        f32x2_split(g[i], g0, g1), f32x2_split(w[i], u0, u1), f32x2_split(v[i], v0, v1);
        v[i] = f32x2(far_gate(g0) ? swiglu_far(g0, u0) : v0, far_gate(g1) ? swiglu_far(g1, u1) : v1);
    }
}

constexpr int kActThreads = 64;  // (small CTAs: 4096 x 14336 SwiGLU 51.5 us with 256 threads, 49.3 with 64; e4m3 quantiser of 16384 x 8192 bf16 77.7 and 71.9)

// The work item of a warp whose lanes have met far gates, from its inputs on, two blocks at a time.  (A function of its own, so that it costs the kernel no registers.)
template <typename T, Out8 OUT>
__device__ __noinline__ void act_block_far(const ActParams p, int64_t row, int col0, int loads)
{
#pragma unroll 1
    for (int u = 0; u < loads; ++u) {
        const int col = col0 + u * 256;
        uint64_t v[1][4];
        act_values_far<T>(act_load<T, true>(p, row, col, col < p.K), v[0]);
        float m[1] = {amax8_nan(v[0])};
        QuantScale qs[1];
        block_scales<OUT, 1>(m, qs);
        out8_store<OUT>(v, qs, [&](int, uint2 w) {
            if (col < p.K) {
                if ((threadIdx.x & 15) == 0) p.s[row * p.KB + (col >> 7)] = qs[0].s;
                *reinterpret_cast<uint2*>(p.q + row * p.K + col) = w;
            }
        });
    }
}

// A scale per 128 columns: sixteen lanes of eight values each.  A work item is 2 LOADS consecutive blocks of a row, for one warp.
template <typename T, bool SWIGLU, Out8 OUT, int LOADS>
__global__ void __launch_bounds__(kActThreads) act_quantize_block_kernel(const ActParams p)
{
    quant_dependency();
    const int lane = threadIdx.x & 31;
    const uint32_t groups = static_cast<uint32_t>((p.KB + 2 * LOADS - 1) / (2 * LOADS));
    const uint32_t item = blockIdx.x * (kActThreads / 32) + (threadIdx.x >> 5);  // the host checks that this fits
    const uint32_t row = item / groups;
    if (row >= p.M) return;  // (a whole warp)
    const int col0 = static_cast<int>(item - row * groups) * (2 * LOADS * 128) + lane * 8;
    ActRaw<T, SWIGLU> raw[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) raw[u] = act_load<T, SWIGLU>(p, row, col0 + u * 256, col0 + u * 256 < p.K);
    uint64_t v[LOADS][4], sums = 0ull;
    float m[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        act_values<T, SWIGLU>(raw[u], v[u], sums);
        m[u] = amax8_nan(v[u]);
    }
    if constexpr (SWIGLU) {
        if (__any_sync(0xffffffffu, act_far(sums))) {
            act_block_far<T, OUT>(p, row, col0, LOADS);
            return;
        }
    }
    QuantScale qs[LOADS];
    block_scales<OUT, LOADS>(m, qs);
    out8_store<OUT>(v, qs, [&](int u, uint2 w) {
        const int col = col0 + u * 256;
        if (col < p.K) {
            if ((lane & 15) == 0) p.s[static_cast<int64_t>(row) * p.KB + (col >> 7)] = qs[u].s;
            *reinterpret_cast<uint2*>(p.q + static_cast<int64_t>(row) * p.K + col) = w;
        }
    });
}

// What a thread of a row with far gates puts right: their values, which the kernel has taken for zeros.  Where one of them may be the row's largest, so that the scale is
// another, or is NaN, the scale becomes NaN, and the row is done again.
template <typename T>
__device__ __noinline__ void swiglu_row_patch(const ActParams p, int64_t row)
{
    const float s = *static_cast<volatile float*>(p.s + row);  // (another thread may be at that)
    bool fits = true;
#pragma unroll 1
    for (int col = threadIdx.x * 8; col < p.K; col += blockDim.x * 8) {
        const T* at = static_cast<const T*>(p.in) + row * 2 * p.K + col;
        uint64_t g[4];
        unpack8<T>(load8(at), g);
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, b;
            f32x2_split(g[i], a, b);
            any |= far_gate(a) || far_gate(b);
        }
        if (!any) continue;
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const float gate = static_cast<float>(at[i]);
            if (!far_gate(gate)) continue;
            const float v = swiglu_far(gate, static_cast<float>(at[p.K + i]));
            if (v == 0.0f) continue;
            // (s is 1 where all other values are zero)
            if (s != 1.0f && fabsf(v) < 126.9f * s) p.q[row * p.K + col + i] = static_cast<uint8_t>(quant_exact(v, s));
            else fits = false;
        }
    }
    if (!fits) *static_cast<volatile float*>(p.s + row) = __int_as_float(0x7fffffff);
}

// A row from its inputs on, by all threads of the CTA, its far gates like the others.
template <typename T>
__device__ __noinline__ void swiglu_row_far(const ActParams p, int64_t row, float* slots)
{
    const int span = blockDim.x * 8;
    float m = 0.0f;
    QuantScale qs{};
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
        for (int col = threadIdx.x * 8; col < p.K; col += span) {
            uint64_t v[4];
            act_values_far<T>(act_load<T, true>(p, row, col, true), v);
            if (pass == 0) m = max_nan(m, amax8_nan(v));
            else *reinterpret_cast<uint2*>(p.q + row * p.K + col) = make_uint2(quant_pack4(v[0], v[1], qs), quant_pack4(v[2], v[3], qs));
        }
        if (pass == 0) {
            __syncwarp();
            m = warp_max_nan(m);
            if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = m;
        }
        __syncthreads();  // (behind the second pass: the slots are free again)
        if (pass == 0) {
            m = (threadIdx.x & 31) < blockDim.x >> 5 ? slots[threadIdx.x & 31] : 0.0f;
            qs = make_out_scale<Out8::kInt8>(warp_max_nan(m));
            if (threadIdx.x == 0) p.s[row] = qs.s;
        }
    }
}

// SwiGLU in int8 with a scale per row: a CTA per row.  Far gates come out as zeros or NaN; rows that have them are put right behind the others, by the threads that
// have met them or, where the scale is NaN or may change, by the CTA.  (A call inside the loop over the rows costs its registers: 4096 x 14336 fp32 99 us for 87,
// bf16 66 for 64.  A call of 16 x 14336 with one such row takes 3 us more, 10 if it is done from its inputs on.)
// LOADS x 8 values a thread stay in registers between the maximum and the quantisation; what lies beyond them is read and computed twice (it hits L2).
template <typename T, int LOADS>
__global__ void __launch_bounds__(1024) swiglu_quantize_row_kernel(const ActParams p)
{
    quant_dependency();
    __shared__ float slots[3][32];
    const int span = blockDim.x * 8, warps = blockDim.x >> 5;
    int parity = 0;
    bool again = false;  // (one flag for all rows: a bit for each is a register more)
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x, parity ^= 1) {
        ActRaw<T, true> raw[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int col = u * span + threadIdx.x * 8;
            raw[u] = act_load<T, true>(p, row, col, col < p.K);
        }
        uint64_t v[LOADS][4], sums = 0ull;
        float m = 0.0f;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            act_values<T, true>(raw[u], v[u], sums);
            m = max_nan(m, amax8_nan(v[u]));
        }
        for (int col = LOADS * span + threadIdx.x * 8; col < p.K; col += span) {
            uint64_t w[4];
            act_values<T, true>(act_load<T, true>(p, row, col, true), w, sums);
            m = max_nan(m, amax8_nan(w));
        }
        again |= act_far(sums);
        m = warp_max_nan(m);
        // (two sets of slots in turn: one barrier per row is enough)
        if ((threadIdx.x & 31) == 0) slots[parity][threadIdx.x >> 5] = m;
        __syncthreads();
        m = (threadIdx.x & 31) < warps ? slots[parity][threadIdx.x & 31] : 0.0f;
        m = warp_max_nan(m);
        const QuantScale qs[1] = {make_out_scale<Out8::kInt8>(m)};
        again |= !(m == m);
        if (threadIdx.x == 0) p.s[row] = qs[0].s;
        uint8_t* q = p.q + row * p.K;
        out8_store<Out8::kInt8>(v, qs, [&](int u, uint2 w) {
            const int col = u * span + threadIdx.x * 8;
            if (col < p.K) *reinterpret_cast<uint2*>(q + col) = w;
        });
        for (int col = LOADS * span + threadIdx.x * 8; col < p.K; col += span) {
            uint64_t w[4];
            act_values<T, true>(act_load<T, true>(p, row, col, true), w, sums);
            *reinterpret_cast<uint2*>(q + col) = make_uint2(quant_pack4(w[0], w[1], qs[0]), quant_pack4(w[2], w[3], qs[0]));
        }
    }
    if (__syncthreads_or(again)) {
        if (again) {
            for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) swiglu_row_patch<T>(p, row);
        }
        __syncthreads();
        for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x)
            if (!(p.s[row] == p.s[row])) swiglu_row_far<T>(p, row, slots[2]);
    }
}

}  // namespace gi8
