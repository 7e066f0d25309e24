// The router of a mixture-of-experts layer: logits [T, E] -> the top_k experts of every token and their weights.
//
//   score  s_e = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   choice c_e = s_e + bias_e;  without a bias l_e itself (s_e increases with it, and l_e needs no rounding)
//   groups: E / G consecutive experts each; a group's value is its largest choice, or the sum of its two largest (of s_e without a
//           bias); the top_groups best groups keep their experts
//   chosen: the top_k largest c_e among them, in that order, the lower index first among equals; c_e = -inf or NaN is never chosen,
//           and where fewer are left the places hold expert -1 and weight 0
//   weight  w_j = s_chosen(j) (/ their sum) * scale
//
// Exactness: which of two experts is chosen must not depend on how a score was rounded to fp32.  The scores are computed in fp32
// together with a bound on their error; a token at which two neighbours in the order (or the last group kept and the first one
// dropped) lie closer than that is decided again in fp64 by the same warp.
//
// One warp per token; a lane holds V consecutive experts, so that the groups of the usual models are runs of whole lanes.
#pragma once

#include <cuda_bf16.h>

#include "../ptx.cuh"

namespace gi8 {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopK = 32;
constexpr int kRouteMaxGroups = 32;

struct RouteParams {
    const void* logits;  // [T, E]
    const float* bias;   // [E] or null
    float* weights;      // [T, k]
    int32_t* experts;    // [T, k]
    int T, E, top_k;
    int groups, top_groups;
    int sigmoid, group_top2, renormalize;
    float scale;
    int vec;             // rows start on whole vectors of a lane's V experts
};

// Order-preserving maps of choices to unsigned keys; 0 for what cannot be chosen.
GI8_DEVICE uint32_t route_key(float c)
{
    if (!(c > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(c + 0.0f);  // -0 becomes +0
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
GI8_DEVICE uint64_t route_key(double c)
{
    if (!(c > -INFINITY)) return 0ull;
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(c + 0.0));
    return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
}
GI8_DEVICE uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
GI8_DEVICE uint64_t warp_max_key(uint64_t k)
{
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
GI8_DEVICE float route_unkey(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
GI8_DEVICE double route_unkey(uint64_t k)
{
    return __longlong_as_double(static_cast<long long>(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}

GI8_DEVICE float route_exp(float x) { return expf(x); }
GI8_DEVICE double route_exp(double x) { return exp(x); }

template <typename F>
struct RouteKeyOf;
template <>
struct RouteKeyOf<float> {
    using type = uint32_t;
};
template <>
struct RouteKeyOf<double> {
    using type = uint64_t;
};

// A group's two largest choices so far (second = -inf: only one).
template <typename F>
GI8_DEVICE void route_two(F c, F& first, F& second)
{
    if (c > first) second = first, first = c;
    else if (c > second) second = c;
}

// The bound on the difference of two fp32 choices' errors, in units of 2^-24.  A score's error: 4 (2 ulp) of the exponential where the score
// moves by at most a quarter of it, 1 for the sum, 4 (2 ulp) for the quotient, 1 for its argument's rounding: 7; softmax: up to V + 5 roundings
// of the denominator's sum and 4 of each exponential instead of the sum's 1: V + 16; the sum with the bias: one rounding of at most |c| + its
// error.  Twice that for the two of them, and half as much again to be safe.
template <int V>
GI8_DEVICE float route_margin(float c, bool softmax) { return (3.0f * 5.9604645e-8f) * (fabsf(c) + (softmax ? V + 16.0f : 8.0f)); }

GI8_DEVICE float route_quotient(float a, float b) { return __fdividef(a, b); }  // 2 ulp for b below 2^126, 0 up to infinity
GI8_DEVICE double route_quotient(double a, double b) { return a / b; }

// Selects one token's experts; the id of place j ends up in lane j.  Returns whether a decision was closer than fp32 can tell
// (F = float only).  l: this lane's logits (-inf behind E).  scratch: E values of this warp.
template <typename F, int V>
GI8_DEVICE bool route_select(const RouteParams& p, const float (&l)[V], F* scratch, int& my_expert, float& row_max, float& denominator)
{
    using Key = typename RouteKeyOf<F>::type;
    const int lane = threadIdx.x & 31;
    const int e0 = lane * V;
    const bool softmax = !p.sigmoid;
    const bool need_scores = p.bias != nullptr || (p.groups > 1 && p.group_top2);
    bool close = false;

    F m = -INFINITY, z = 0;
    if (softmax && (need_scores || !p.renormalize)) {
        float mm = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) mm = fmaxf(mm, l[i]);
        const uint32_t mk = __reduce_max_sync(0xffffffffu, route_key(mm));
        m = mk ? static_cast<F>(route_unkey(mk)) : F(0);
#pragma unroll
        for (int i = 0; i < V; ++i) z += l[i] > -INFINITY ? route_exp(static_cast<F>(l[i]) - m) : F(0);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        row_max = static_cast<float>(m), denominator = static_cast<float>(z);
    }
    auto score = [&](float v) -> F {
        if (!(v > -INFINITY)) return F(0);
        return softmax ? route_quotient(route_exp(static_cast<F>(v) - m), z) : route_quotient(F(1), F(1) + route_exp(-static_cast<F>(v)));
    };

    F c[V];
    F first = -INFINITY, second = -INFINITY;  // of this lane's choices, as far as groups need them
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const bool masked = !(l[i] > -INFINITY);
        const F s = need_scores && !masked ? score(l[i]) : F(0);
        const F choice = p.bias ? s + static_cast<F>(e0 + i < p.E ? __ldg(p.bias + e0 + i) : 0.0f) : static_cast<F>(l[i]);
        c[i] = masked || !(choice > -INFINITY) ? F(-INFINITY) : choice;
        const F of_group = masked ? F(-INFINITY) : (p.group_top2 && !p.bias) ? s : c[i];
        if (p.groups > 1) route_two(of_group, first, second);
        if (p.groups > 1 && scratch && e0 + i < p.E) scratch[e0 + i] = of_group;
    }

    if (p.groups > 1) {
        const int size = p.E / p.groups;
        int group_here;  // the group whose value this lane holds
        bool holds = true;
        if (!scratch) {  // whole lanes, a power of two of them
            const int span = size / V;
            group_here = lane >> (__ffs(span) - 1);
            holds = group_here < p.groups;
            for (int o = 1; o < span; o <<= 1) {
                const F f2 = __shfl_xor_sync(0xffffffffu, first, o), s2 = __shfl_xor_sync(0xffffffffu, second, o);
                route_two(f2, first, second);
                route_two(s2, first, second);
            }
        } else {
            __syncwarp();
            group_here = lane;
            holds = lane < p.groups;
            first = second = -INFINITY;
            if (holds)
                for (int i = 0; i < size; ++i) route_two(scratch[lane * size + i], first, second);
            __syncwarp();
        }
        const F value = p.group_top2 && second > -INFINITY ? first + second : first;
        Key key = holds ? route_key(value) : Key(0);
        uint32_t kept = 0;
        F last = 0;
        for (int n = 0; n <= p.top_groups; ++n) {
            const Key best = warp_max_key(key);
            if (best == 0) break;
            const int src = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
            const int g = __shfl_sync(0xffffffffu, group_here, src);
            if (n == p.top_groups) {  // the best one that stays out
                if (need_scores && last - route_unkey(best) <= 2 * route_margin<V>(static_cast<float>(last), softmax)) close = true;
                break;
            }
            last = route_unkey(best);
            kept |= 1u << g;
            if (group_here == g) key = 0;
        }
        if (!scratch) {  // a lane's experts are of one group
            const bool out = holds && !((kept >> group_here) & 1u);
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = out ? F(-INFINITY) : c[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int g = (e0 + i) / size;
                if (g < p.groups && !((kept >> g) & 1u)) c[i] = -INFINITY;
            }
        }
    }

    Key key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = route_key(c[i]);
    my_expert = -1;
    F last = 0;
    const int rounds = p.top_k + (p.bias ? 1 : 0);  // one more to see how far the first one left out is
    for (int j = 0; j < rounds; ++j) {
        Key best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = max(best, key[i]);
        const Key top = warp_max_key(best);
        if (top == 0) break;
        if (p.bias) {
            const F here = route_unkey(top);
            if (j > 0 && last - here <= route_margin<V>(static_cast<float>(last), softmax)) close = true;
            last = here;
        }
        if (j == p.top_k) break;
        // the first lane that has it, and its first
        const int src = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
        int at = 0;
        bool looking = lane == src;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const bool hit = looking && key[i] == top;
            key[i] = hit ? Key(0) : key[i];
            at = hit ? i : at;
            looking = looking && !hit;
        }
        const int e = __shfl_sync(0xffffffffu, e0 + at, src);
        my_expert = lane == j ? e : my_expert;
    }
    return close;
}

GI8_DEVICE float route_load(const float* p) { return __ldg(p); }
GI8_DEVICE float route_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }

template <typename T, int V>
GI8_DEVICE void route_load_lane(const T* row, int e0, int E, bool vec, float (&l)[V])
{
    constexpr int kBytes = V * static_cast<int>(sizeof(T));
    if constexpr (kBytes % 16 == 0) {
        if (vec) {
            if (e0 < E) {
                constexpr int kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
                for (int i = 0; i < V; i += kPer) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + e0 + i));
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (sizeof(T) == 4) {
                            l[i + j] = __uint_as_float(w[j]);
                        } else {
                            l[i + 2 * j] = __uint_as_float(w[j] << 16);
                            l[i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) l[i] = -INFINITY;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = e0 + i < E ? route_load(row + e0 + i) : -INFINITY;
}

template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_experts_kernel(const RouteParams p, int use_scratch)
{
    extern __shared__ double route_scratch[];  // use_scratch: E values per warp
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
    if (t >= p.T) return;
    const T* row = static_cast<const T*>(p.logits) + t * p.E;
    float l[V];
    route_load_lane<T, V>(row, lane * V, p.E, p.vec, l);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (!(l[i] > -INFINITY)) l[i] = -INFINITY;  // NaN is never chosen

    int expert;
    float row_max = 0.0f, denominator = 1.0f;
    double* mine = use_scratch ? route_scratch + static_cast<int64_t>(warp) * p.E : nullptr;
    if (route_select<float, V>(p, l, reinterpret_cast<float*>(mine), expert, row_max, denominator))
        route_select<double, V>(p, l, mine, expert, row_max, denominator);

    // Weights, lane j those of place j.  Their ratios do not depend on the softmax's denominator, nor on the sigmoid's where it is
    // all but exp(l): renormalised weights are taken relative to the largest logit chosen, so that they never are 0 / 0.
    const bool chosen = lane < p.top_k && expert >= 0;
    const float v = chosen ? route_load(row + expert) : -INFINITY;
    float top = v;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float w = 0.0f;
    if (chosen) {
        if (!p.sigmoid) w = p.renormalize ? expf(v - top) : expf(v - row_max) / denominator;
        else if (p.renormalize && top < -80.0f) w = expf(v - top);
        else w = 1.0f / (1.0f + expf(-v));
    }
    if (p.renormalize) {
        float sum = w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (chosen) w /= sum;
    }
    if (lane < p.top_k) {
        p.weights[t * p.top_k + lane] = w * p.scale;
        p.experts[t * p.top_k + lane] = expert;
    }
}

}  // namespace gi8
