// Elementwise activations in 8 bits: the e4m3 quantiser, and SwiGLU behind the product of gate and up rows,
//   v = g / (1 + exp(-g)) u   of the two halves of a row,   in fp32 from fp32 or bf16,
// with a scale per row and 128 columns, or (SwiGLU in int8) one per row.  Every element is read and written once.  Bound: HBM, with instruction issue close behind for
// bf16 input: SwiGLU 4096 x 14336 48 us, 6.15 TB/s (0.94 of the copy rate; 17.7 instructions an element issued on 65 % of the cycles), fp32 78 us, 6.8 TB/s; e4m3
// quantiser 16384 x 8192 bf16 72 us, 5.7 TB/s, fp32 98 us, 6.9 TB/s; per row 4096 x 14336 62 us, 4.7 TB/s (a CTA's loads, maximum and stores follow each other; two
// CTAs of 448 threads share an SM).
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

// g u / (1 + 2^(-g log2 e)) for a pair, in packed steps but for the exponentials and reciprocals, which the special-function unit takes one by one
// (subnormal results flushed: next to 1 they are nothing, and a reciprocal of 2^126 and more, or of an overflowed exponential, is the limit 0).
// Good to (5 + |g|) units in the last place, next to the half step of 1/254 or 2^-4 that the result is rounded by.
// (Of 63 million e4m3 results of fp32 input 47 lay on the other side of a rounding step than the exact ones; of the same sum with expf and a division 43, of torch's silu
// 52.  Those took 129 us for 96 with a scale per row, 4096 x 14336, and the same with block scales.)
GI8_DEVICE uint64_t swiglu2(uint64_t g, uint64_t u)
{
    float a, b;
    f32x2_split(mul2(g, f32x2(-1.44269504f, -1.44269504f)), a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    f32x2_split(add2(f32x2(a, b), f32x2(1.0f, 1.0f)), a, b);
    return mul2(mul2(g, f32x2(approx_reciprocal(a), approx_reciprocal(b))), u);
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
GI8_DEVICE void act_values(const ActRaw<T, SWIGLU>& r, uint64_t (&v)[4])
{
    unpack8<T>(r.a, v);
    if constexpr (SWIGLU) {
        uint64_t w[4];
        unpack8<T>(r.b, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = swiglu2(v[i], w[i]);
    }
}

constexpr int kActThreads = 64;  // (small CTAs: 4096 x 14336 SwiGLU 51.5 us with 256 threads, 49.3 with 64; e4m3 quantiser of 16384 x 8192 bf16 77.7 and 71.9)

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
    uint64_t v[LOADS][4];
    float m[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
        act_values<T, SWIGLU>(raw[u], v[u]);
        m[u] = amax8_nan(v[u]);
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

// SwiGLU in int8 with a scale per row: a CTA per row.  LOADS x 8 values a thread stay in registers between the maximum and the quantisation;
// what lies beyond them is read and computed twice (it hits L2).
template <typename T, int LOADS>
__global__ void __launch_bounds__(1024) swiglu_quantize_row_kernel(const ActParams p)
{
    quant_dependency();
    __shared__ float slots[2][32];
    const int span = blockDim.x * 8, warps = blockDim.x >> 5;
    int parity = 0;
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x, parity ^= 1) {
        ActRaw<T, true> raw[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int col = u * span + threadIdx.x * 8;
            raw[u] = act_load<T, true>(p, row, col, col < p.K);
        }
        uint64_t v[LOADS][4];
        float m = 0.0f;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            act_values<T, true>(raw[u], v[u]);
            m = max_nan(m, amax8_nan(v[u]));
        }
        for (int col = LOADS * span + threadIdx.x * 8; col < p.K; col += span) {
            uint64_t w[4];
            act_values<T, true>(act_load<T, true>(p, row, col, true), w);
            m = max_nan(m, amax8_nan(w));
        }
        m = warp_max_nan(m);
        // (two sets of slots in turn: one barrier per row is enough)
        if ((threadIdx.x & 31) == 0) slots[parity][threadIdx.x >> 5] = m;
        __syncthreads();
        m = (threadIdx.x & 31) < warps ? slots[parity][threadIdx.x & 31] : 0.0f;
        const QuantScale qs[1] = {make_out_scale<Out8::kInt8>(warp_max_nan(m))};
        if (threadIdx.x == 0) p.s[row] = qs[0].s;
        uint8_t* q = p.q + row * p.K;
        out8_store<Out8::kInt8>(v, qs, [&](int u, uint2 w) {
            const int col = u * span + threadIdx.x * 8;
            if (col < p.K) *reinterpret_cast<uint2*>(q + col) = w;
        });
        for (int col = LOADS * span + threadIdx.x * 8; col < p.K; col += span) {
            uint64_t w[4];
            act_values<T, true>(act_load<T, true>(p, row, col, true), w);
            *reinterpret_cast<uint2*>(q + col) = make_uint2(quant_pack4(w[0], w[1], qs[0]), quant_pack4(w[2], w[3], qs[0]));
        }
    }
}

}  // namespace gi8
