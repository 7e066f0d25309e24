// out[t, n] = bf16( add[t, n] + sum_j weights[t, j] * y[places[t, j], n] ): one fused multiply-add in fp32 per choice, ascending j,
// starting from `add` (or zero); choices without a place are left out.  Bound by HBM: k rows read, one written per token.
#pragma once

#include "../ptx.cuh"

namespace gi8 {

constexpr int kCombineThreads = 256;
constexpr int kCombineMaxTopK = 32;

struct CombineParams {
    const uint16_t* y;      // bf16 [rows, N]
    const float* weights;   // [T, k]
    const int32_t* places;  // [T, k]
    const void* add;        // fp32 or bf16 [T, N], or null
    uint16_t* out;          // bf16 [T, N]
    int64_t rows;
    int T, N, top_k;
};

// VEC columns per thread: 8 (16-byte accesses) or 1.  ADD_F32: `add` is fp32 and starts the sum as it is.
template <int VEC, bool ADD_F32>
__global__ void __launch_bounds__(kCombineThreads)
combine_experts_kernel(const CombineParams p)
{
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t t = blockIdx.x;
    const int64_t col = (static_cast<int64_t>(blockIdx.y) * kCombineThreads + threadIdx.x) * VEC;
    int my_place = -1;
    float my_weight = 0.0f;
    if (lane < p.top_k) {
        my_place = __ldg(p.places + t * p.top_k + lane);
        my_weight = __ldg(p.weights + t * p.top_k + lane);
        if (my_place >= p.rows) my_place = -1;
    }
    const bool live = col < p.N;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    auto load = [&](const uint16_t* base, uint32_t (&w)[(VEC + 1) / 2]) {
        if constexpr (VEC == 8) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(base));
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        } else {
            w[0] = __ldg(base);
        }
    };
    if (live && p.add) {
        const int64_t at = t * p.N + col;
        if constexpr (ADD_F32) {
            const float* add = static_cast<const float*>(p.add) + at;
            if constexpr (VEC == 8) {
                const float4 lo = __ldg(reinterpret_cast<const float4*>(add)), hi = __ldg(reinterpret_cast<const float4*>(add) + 1);
                acc[0] = lo.x, acc[1] = lo.y, acc[2] = lo.z, acc[3] = lo.w, acc[4] = hi.x, acc[5] = hi.y, acc[6] = hi.z, acc[7] = hi.w;
            } else {
                acc[0] = __ldg(add);
            }
        } else {
            uint32_t w[(VEC + 1) / 2];
            load(static_cast<const uint16_t*>(p.add) + at, w);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = __uint_as_float((i & 1) ? (w[i / 2] & 0xffff0000u) : (w[i / 2] << 16));
        }
    }
    constexpr int kAhead = 4;  // rows requested together
    for (int j0 = 0; j0 < p.top_k; j0 += kAhead) {
        uint32_t w[kAhead][(VEC + 1) / 2];
        int place[kAhead];
        float weight[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            place[j] = __shfl_sync(0xffffffffu, my_place, (j0 + j) & 31);
            weight[j] = __shfl_sync(0xffffffffu, my_weight, (j0 + j) & 31);
            if (j0 + j >= p.top_k) place[j] = -1;
            if (live && place[j] >= 0) load(p.y + static_cast<int64_t>(place[j]) * p.N + col, w[j]);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (place[j] >= 0) {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    acc[i] = fmaf(weight[j], __uint_as_float((i & 1) ? (w[j][i / 2] & 0xffff0000u) : (w[j][i / 2] << 16)), acc[i]);
            }
    }
    if (!live) return;
    uint16_t* dst = p.out + t * p.N + col;
    if constexpr (VEC == 8) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]), pack_bf16x2(acc[4], acc[5]), pack_bf16x2(acc[6], acc[7]));
    } else {
        *dst = to_bf16_bits(acc[0]);
    }
}

}  // namespace gi8
