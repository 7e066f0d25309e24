// The router of a mixture-of-experts layer: logits [T, E] -> the top_k experts of every token and their weights.
//
//   score  s_e = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   choice c_e = s_e + bias_e;  without a bias l_e itself (s_e increases with it, and l_e needs no rounding)
//   groups: E / G consecutive experts each; a group's value is its largest choice, or the sum of its two largest (of s_e without a
//           bias); the top_groups best groups keep their experts
//           (l_e = +inf counts as the largest finite value: a softmax shares its weight among the infinite ones)
//   chosen: the top_k largest c_e among them, in that order, the lower index first among equals; c_e = -inf or NaN is never chosen,
//           and where fewer are left the places hold expert -1 and weight 0
//   weight  w_j = s_chosen(j) (/ their sum) * scale
//
// Exactness: which of two experts is chosen must not depend on how a score was rounded to fp32: what is equal in fp64 is equal, and nothing else.
// A token is decided by fp32 scores, with a bound on their error.  Where two neighbours in the order, or a group kept and one dropped, lie closer
// than that, the token is marked and decided again behind the loop over the warp's tokens: the groups' values in fp64, and the candidates,
// which are those chosen and what lies as close behind them, put in order by their choices in fp64, a lane each.  Of tokens whose logits are
// spread over all of fp32 one in a thousand or so comes there, and the warp that it holds up may be the launch's last: what counts is how long
// it takes (all of a token's scores in fp64 and the whole selection again took 13 us, and the launch of 16384 tokens 39), and that it costs the
// other tokens no registers.  Equal fp32 logits are marked as well: 16384 tokens whose 256 fp32 logits hold bf16 values take 30 us for 14.9 (as
// bf16 tensors, whose keys lose nothing, 13.4).
//
// One warp per token; a lane holds V consecutive experts, so that the groups of the usual models are runs of whole lanes.  The choices become
// unsigned keys whose lowest bits are the place within the lane, sorted in every lane, so that a round of the selection is one maximum over
// the lanes' first keys and a shift of the winner's lane.  Up to four tokens' weights (eight experts each) are made together, a lane each.
// Bound by instruction issue and latencies: 16384 tokens of 256 experts, bias, groups 25.7 us (890 instructions a token, issued in 60 % of
// the cycles; 1735 and 38 us with whole choices and indices apart), of which the bytes take 2.7; the selection alone, without bias and groups,
// 14.9; 16 tokens 3.9, of which an empty launch takes 1.8.
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
    int vec, vec_bias;   // rows (the bias) can be read in 16-byte pieces of a lane's V experts
    int half_k;          // half of the power of two that holds top_k (0: one)
    int batch;           // tokens that a warp decides before it makes their weights together, at most 32 / that power of two
};

// Order-preserving map of choices to unsigned keys.  What cannot be chosen is -inf, whose key is kRouteNone.
constexpr uint32_t kRouteNone = 0x007fffffu;
GI8_DEVICE uint32_t route_key(float c)
{
    const uint32_t u = __float_as_uint(c + 0.0f);  // -0 becomes +0
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
GI8_DEVICE float route_unkey(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
GI8_DEVICE uint64_t route_key(double c)  // 0: cannot be chosen
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

// A group's two largest choices so far (second = -inf: only one).
template <typename F>
GI8_DEVICE void route_two(F c, F& first, F& second)
{
    second = max(second, min(first, c));
    first = max(first, c);
}

// The largest and second largest of a group's choices, in every lane of the group (whole lanes, a power of two of them) or, through shared
// memory, in lane g for group g.  first, second: of this lane's choices.  Returns the group whose values the lane holds, or -1.
template <typename F, int V>
GI8_DEVICE int route_group_best(const RouteParams& p, const F (&of_group)[V], F* scratch, F& first, F& second)
{
    const int lane = threadIdx.x & 31;
    const int size = p.E / p.groups;
    first = second = -INFINITY;
    if (!scratch) {
#pragma unroll
        for (int i = 0; i < V; ++i) route_two(of_group[i], first, second);
        const int span = size / V;
        for (int o = 1; o < span; o <<= 1) {
            const F f2 = __shfl_xor_sync(0xffffffffu, first, o), s2 = __shfl_xor_sync(0xffffffffu, second, o);
            second = max(max(second, s2), min(first, f2));
            first = max(first, f2);
        }
        const int g = lane >> (__ffs(span) - 1);
        return g < p.groups ? g : -1;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (lane * V + i < p.E) scratch[lane * V + i] = of_group[i];
    __syncwarp();
    if (lane < p.groups)
        for (int i = 0; i < size; ++i) route_two(scratch[lane * size + i], first, second);
    return lane < p.groups ? lane : -1;
}

// Takes the experts of the groups that are not kept out of the choice.  group_here: what route_group_best returned.
template <typename F, int V>
GI8_DEVICE void route_drop_groups(const RouteParams& p, uint32_t kept, int group_here, bool by_lane, F (&c)[V])
{
    if (by_lane) {
        const bool out = group_here >= 0 && !((kept >> group_here) & 1u);
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = out ? F(-INFINITY) : c[i];
    } else {
        const int size = p.E / p.groups, e0 = (threadIdx.x & 31) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int g = (e0 + i) / size;
            if (g < p.groups && !((kept >> g) & 1u)) c[i] = -INFINITY;
        }
    }
}

// A bound on the difference of two fp32 scores' errors, in units of 2^-24, where the choice is by scores.  Sigmoid: the exponential's (2 + 1.173
// |l|) ulp move the score by at most 1/4, and by less far out: 1.6; the sum 1 (times a quarter), the reciprocal 2 (1 ulp): below 7.  Softmax: 5
// for the score's own exponential and 4 for the quotient, the denominator's sum V + 5 and its exponentials 4: below V + 20.  The bias is
// added with one rounding, of at most |c|.  Twice that for the two of them, and half as much again to be safe.
template <int V>
GI8_DEVICE float route_margin(float c, bool softmax) { return (3.0f * 5.9604645e-8f) * (fabsf(c) + (softmax ? V + 21.0f : 8.0f)); }

// A group's fp32 value.  A sum of two largest choices is halved, as all of them are: two finite choices can be beyond fp32 together.
GI8_DEVICE float route_group_value(const RouteParams& p, float first, float second)
{
    return !p.group_top2 ? first : second > -INFINITY ? 0.5f * first + 0.5f * second : 0.5f * first;
}

// A bound on its error (three times what a choice is off by, for each of those that it is made of; the sum's own rounding is at most theirs).
// It goes by the choices' magnitudes and not by the value's: choices of opposite signs cancel, their errors do not.
template <int V>
GI8_DEVICE float route_group_slack(const RouteParams& p, float first, float second, bool softmax)
{
    if (!p.group_top2) return route_margin<V>(first, softmax);
    return 0.5f * route_margin<V>(fabsf(first) + (second > -INFINITY ? fabsf(second) : 0.0f), softmax);  // (infinite: fp64 decides)
}

// Whole warp: may a group that is dropped be ahead of one that is kept?  value, slack: of the lane's group, where it is live (has a choice).
GI8_DEVICE bool route_groups_close(float value, float slack, bool live, bool kept)
{
    const uint32_t low = __reduce_min_sync(0xffffffffu, kept ? route_key(value - slack) : 0xffffffffu);
    const uint32_t high = __reduce_max_sync(0xffffffffu, live && !kept ? route_key(value + slack) : 0u);
    return high != 0 && high >= low;
}

// The softmax's largest logit and denominator (0 and 0 for a row without logits), in fp32 or fp64.
template <typename F, int V>
GI8_DEVICE void route_denominator(const float (&l)[V], F& m, F& z)
{
    float mm = l[0];
#pragma unroll
    for (int i = 1; i < V; ++i) mm = fmaxf(mm, l[i]);
    mm = route_unkey(warp_max_key(route_key(mm)));
    m = mm > -INFINITY ? static_cast<F>(mm) : F(0);
    z = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) z += exp(static_cast<F>(l[i]) - m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
}

// Descending order within a lane: Batcher's merge exchange sort, unrolled.
template <int V>
GI8_DEVICE void route_sort(uint32_t (&key)[V])
{
#pragma unroll
    for (int p = 1; p < V; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t hi = max(key[i + j], key[i + j + k]), lo = min(key[i + j], key[i + j + k]);
                        key[i + j] = hi, key[i + j + k] = lo;
                    }
}

GI8_DEVICE float route_load(const float* p) { return __ldg(p); }
GI8_DEVICE float route_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// A logit as it counts: NaN as -inf, +inf as the largest finite value (a softmax of it is finite then).
GI8_DEVICE float route_logit(float l) { return fminf(fmaxf(l, -INFINITY), 3.402823466e38f); }

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

// The groups that are kept, in fp64 (groups of whole lanes).
template <int V>
GI8_DEVICE uint32_t route_groups_exact(const RouteParams& p, const float (&l)[V], const float (&bias)[V])
{
    const bool softmax = !p.sigmoid, scores = p.bias || p.group_top2;
    double m = 0.0, z = 1.0;
    if (softmax && scores) route_denominator(l, m, z);
    double of_group[V], first, second;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        double v = static_cast<double>(l[i]);
        if (scores) {
            const double x = exp(softmax ? v - m : -v);
            v = softmax ? x / z : 1.0 / (1.0 + x);
        }
        if (p.bias) v += static_cast<double>(bias[i]);
        of_group[i] = l[i] > -INFINITY && v > -INFINITY ? v : -INFINITY;
    }
    const int group_here = route_group_best(p, of_group, static_cast<double*>(nullptr), first, second);
    uint64_t key = group_here >= 0 ? route_key(p.group_top2 && second > -INFINITY ? first + second : first) : 0ull;
    uint32_t kept = 0;
    for (int n = 0; n < p.top_groups; ++n) {
        const uint64_t best = warp_max_key(key);
        if (best == 0) break;
        const int g = __shfl_sync(0xffffffffu, group_here, __ffs(__ballot_sync(0xffffffffu, key == best)) - 1);
        kept |= 1u << g;
        if (group_here == g) key = 0;
    }
    return kept;
}

// The candidates e of lanes 0 .. n - 1, put in descending order of their choices in fp64, the lower index first among equals.
template <typename T, int V>
GI8_DEVICE int route_order_exact(const RouteParams& p, const float (&l)[V], const T* row, int e, int n)
{
    const int lane = threadIdx.x & 31;
    const bool softmax = !p.sigmoid;
    double m = 0.0, z = 1.0;
    if (softmax && p.bias) route_denominator(l, m, z);
    double c = lane < n ? static_cast<double>(route_logit(route_load(row + e))) : 0.0;
    if (p.bias && lane < n) {
        const double x = exp(softmax ? c - m : -c);
        c = (softmax ? x / z : 1.0 / (1.0 + x)) + static_cast<double>(__ldg(p.bias + e));
    }
    int rank = 0;
    for (int i = 0; i < n; ++i) {
        const double ci = __shfl_sync(0xffffffffu, c, i);
        const int ei = __shfl_sync(0xffffffffu, e, i);
        rank += ci > c || (ci == c && ei < e);
    }
    int mine = -1;
    for (int i = 0; i < n; ++i) {
        const int r = __shfl_sync(0xffffffffu, rank, i), ei = __shfl_sync(0xffffffffu, e, i);
        mine = r == lane ? ei : mine;
    }
    return mine;
}

// One token by fp32 keys; the expert of place j ends up in lane j, -1 for none.
// l: this lane's logits (-inf behind E and for NaN).
// Returns true where the candidates are more than there are lanes, or the groups' values too close and not to be had from lanes.
template <typename T, int V>
GI8_DEVICE bool route_fast(const RouteParams& p, const T* row, const float (&l)[V], const float (&bias)[V], float* scratch, float row_max, float denominator, int& my_expert)
{
    constexpr uint32_t kPlace = V <= 1 ? 0u : V <= 2 ? 1u : V <= 4 ? 3u : V <= 8 ? 7u : V <= 16 ? 15u : 31u;
    const int lane = threadIdx.x & 31;
    const bool softmax = !p.sigmoid;
    const bool scores_of_groups = p.groups > 1 && p.group_top2;
    const bool by_scores = p.bias != nullptr;
    bool close = false;
    float c[V];
    auto score = [&](float v) { return softmax ? __fdividef(expf(v - row_max), denominator) : approx_reciprocal(1.0f + __expf(-v)); };
#pragma unroll
    for (int i = 0; i < V; ++i) {
        c[i] = l[i];
        if (by_scores) c[i] = l[i] > -INFINITY ? fmaxf(score(l[i]) + bias[i], -INFINITY) : -INFINITY;
    }
    if (p.groups > 1) {
        float of_group[V], first, second;
#pragma unroll
        for (int i = 0; i < V; ++i) of_group[i] = scores_of_groups && !by_scores && l[i] > -INFINITY ? score(l[i]) : c[i];
        const int group_here = route_group_best(p, of_group, scratch, first, second);
        const float value = route_group_value(p, first, second);
        uint32_t key = group_here >= 0 ? route_key(value) : 0u;
        uint32_t kept = 0;
        for (int n = 0; n < p.top_groups; ++n) {
            const uint32_t best = warp_max_key(key);
            if (best <= kRouteNone) break;
            const int g = __shfl_sync(0xffffffffu, group_here, __ffs(__ballot_sync(0xffffffffu, key == best)) - 1);
            kept |= 1u << g;
            if (group_here == g) key = 0;
        }
        if (by_scores || scores_of_groups) {
            const bool live = group_here >= 0 && value > -INFINITY;
            close = route_groups_close(value, route_group_slack<V>(p, first, second, softmax), live, live && ((kept >> group_here) & 1u));
        }
        if (close) {  // (the same in all lanes)
            if (scratch) return true;
            kept = route_groups_exact(p, l, bias);
            close = false;
        }
        route_drop_groups(p, kept, group_here, !scratch, c);
    }
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = (route_key(c[i]) & ~kPlace) | (kPlace - i);
    route_sort(key);
    uint32_t mine = 0;
    int found = 0;
    my_expert = -1;
    // Takes the largest key that is left; false: nobody can be chosen any more.
    auto take = [&]() {
        const uint32_t top = warp_max_key(key[0]);
        if (top <= kRouteNone) return false;
        // the first lane that has this value, and the first place there
        const int src = __ffs(__ballot_sync(0xffffffffu, (key[0] | kPlace) == (top | kPlace))) - 1;
        const uint32_t taken = __shfl_sync(0xffffffffu, key[0], src);
        mine = lane == found ? taken : mine;
        my_expert = lane == found ? src * V + static_cast<int>(kPlace - (taken & kPlace)) : my_expert;
        const bool next = lane == src;
#pragma unroll
        for (int i = 0; i + 1 < V; ++i) key[i] = next ? key[i + 1] : key[i];
        key[V - 1] = next ? 0u : key[V - 1];
        ++found;
        return true;
    };
    for (int j = 0; j < p.top_k; ++j)
        if (!take()) break;
    {
        // Neighbours in the order, the first one left out among them; what keys drop below a value is at most their lowest bits' worth of it.
        auto bound = [&](float a, float b) {
            const float lost = (kPlace + 1) * 1.1920929e-7f * fmaxf(fabsf(a), fabsf(b));
            return by_scores ? route_margin<V>(a, softmax) + lost : lost;
        };
        const uint32_t left = warp_max_key(key[0]);
        uint32_t after = __shfl_down_sync(0xffffffffu, mine, 1);
        if (lane == found - 1) after = left;
        if (lane < found && after > kRouteNone) {
            const float a = route_unkey(mine & ~kPlace), b = route_unkey(after & ~kPlace);
            close = a - b <= bound(a, b);
        }
        if (__any_sync(0xffffffffu, close)) {
            const float last = route_unkey(__shfl_sync(0xffffffffu, mine, found - 1) & ~kPlace);
            while (true) {
                const uint32_t top = warp_max_key(key[0]);
                if (top <= kRouteNone) break;
                const float b = route_unkey(top & ~kPlace);
                if (last - b > bound(last, b)) break;
                if (found == 32) return true;
                take();
            }
            my_expert = route_order_exact(p, l, row, my_expert, found);
        }
    }
    if (lane >= p.top_k) my_expert = -1;
    return false;
}

// The same in fp64 from the start, for what is left: through shared memory (E values of the warp) and in loops, so that it costs the
// others neither registers nor room for instructions.
template <typename T, int V>
GI8_DEVICE int route_exact(const RouteParams& p, const T* row, double* c)
{
    const int lane = threadIdx.x & 31;
    const bool softmax = !p.sigmoid;
    const bool scores_of_groups = p.groups > 1 && p.group_top2 && !p.bias;
    double m = -INFINITY, z = 0.0;
    if (softmax) {
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32) m = fmax(m, static_cast<double>(route_logit(route_load(row + e))));
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!(m > -INFINITY)) m = 0.0;
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32) {
            const float l = route_logit(route_load(row + e));
            if (l > -INFINITY) z += exp(static_cast<double>(l) - m);
        }
#pragma unroll 1
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    // Choices, or first the scores that the groups' values are sums of.
    auto fill = [&](bool scores, bool bias) {
        __syncwarp();
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32) {
            const double l = static_cast<double>(route_logit(route_load(row + e)));
            double v = l;
            if (scores) {
                const double x = exp(softmax ? l - m : -l);
                v = (softmax ? x : 1.0) / (softmax ? z : 1.0 + x);
            }
            if (bias) v += static_cast<double>(__ldg(p.bias + e));
            c[e] = l > -INFINITY && v > -INFINITY ? v : -INFINITY;
        }
        __syncwarp();
    };
    const bool by_scores = p.bias != nullptr;
    uint32_t kept = 0xffffffffu;
    const int size = p.E / p.groups;
    if (p.groups > 1) {
        fill(by_scores || scores_of_groups, by_scores);
        double first = -INFINITY, second = -INFINITY;
        if (lane < p.groups)
#pragma unroll 1
            for (int i = 0; i < size; ++i) route_two(c[lane * size + i], first, second);
        uint64_t key = route_key(p.group_top2 && second > -INFINITY ? first + second : first);
        kept = 0;
#pragma unroll 1
        for (int n = 0; n < p.top_groups; ++n) {
            const uint64_t best = warp_max_key(key);
            if (best == 0) break;
            const int g = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
            kept |= 1u << g;
            if (lane == g) key = 0;
        }
    }
    if (p.groups == 1 || (scores_of_groups && !by_scores)) fill(by_scores, by_scores);
    int my_expert = -1;
#pragma unroll 1
    for (int j = 0; j < p.top_k; ++j) {
        uint64_t best = 0;
        int at = 0;
#pragma unroll 1
        for (int e = lane * V; e < min((lane + 1) * V, p.E); ++e) {
            const uint64_t key = (kept >> (e / size)) & 1u ? route_key(c[e]) : 0ull;
            if (key > best) best = key, at = e;
        }
        const uint64_t top = warp_max_key(best);
        if (top == 0) break;
        const int src = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
        const int e = __shfl_sync(0xffffffffu, at, src);
        my_expert = lane == j ? e : my_expert;
        if (lane == src) c[e] = -INFINITY;
        __syncwarp();
    }
    return my_expert;
}

// A token by the careful way, from its logits on.
template <typename T, int V>
GI8_DEVICE int route_carefully(const RouteParams& p, const T* row, double* scratch, int use_scratch, float& m, float& z)
{
    const int lane = threadIdx.x & 31;
    float l[V], bias[V];
    route_load_lane<T, V>(row, lane * V, p.E, p.vec, l);
    if (p.bias) route_load_lane<float, V>(p.bias, lane * V, p.E, p.vec_bias, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = route_logit(l[i]);
    m = 0.0f, z = 1.0f;
    if (!p.sigmoid && (p.bias || !p.renormalize || (p.groups > 1 && p.group_top2))) route_denominator(l, m, z);
    int expert;
    if (route_fast<T, V>(p, row, l, bias, use_scratch ? reinterpret_cast<float*>(scratch) : nullptr, m, z, expert)) expert = route_exact<T, V>(p, row, scratch);
    return expert;
}

template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32, V <= 8 ? 8 : 3)
route_experts_kernel(const __grid_constant__ RouteParams p, int use_scratch)
{
    extern __shared__ double route_scratch[];  // E values per warp
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    constexpr uint32_t kPlace = V <= 1 ? 0u : V <= 2 ? 1u : V <= 4 ? 3u : V <= 8 ? 7u : V <= 16 ? 15u : 31u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    double* exact_c = route_scratch + warp * p.E;
    float* scratch = use_scratch ? reinterpret_cast<float*>(exact_c) : nullptr;
    const bool softmax = !p.sigmoid, by_scores = p.bias != nullptr;
    const bool scores_of_groups = p.groups > 1 && p.group_top2 && !by_scores;
    const bool need_denominator = softmax && (by_scores || scores_of_groups || !p.renormalize);
    // Equal keys mean equal logits where the bits that keys lose are zeros in all of them.
    const bool exact = sizeof(T) == 2 && !by_scores;
    const int wide = p.half_k > 0 ? 2 * p.half_k : 1;  // lanes of a token's places
    const int my_slot = lane / wide, my_place = lane - my_slot * wide;
    float bias[V];
    if (by_scores) route_load_lane<float, V>(p.bias, lane * V, p.E, p.vec_bias, bias);

    // Weights, by the lanes of a token's places.  Their ratios do not depend on the softmax's denominator, nor on the sigmoid's where it is all
    // but exp(l): renormalised weights are taken relative to the largest logit chosen, so that they never are 0 / 0.
    auto finish = [&](int64_t t, bool token, int expert, float row_max, float denominator) {
        const bool chosen = token && my_place < p.top_k && expert >= 0;
        const float v = chosen ? route_logit(route_load(static_cast<const T*>(p.logits) + t * p.E + expert)) : -INFINITY;
        float top = v;
        for (int o = p.half_k; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float w = 0.0f;
        if (chosen) {
            if (softmax) w = p.renormalize ? expf(v - top) : __fdividef(expf(v - row_max), denominator);
            else if (p.renormalize && top < -80.0f) w = expf(v - top);
            else w = __fdividef(1.0f, 1.0f + expf(-v));
        }
        if (p.renormalize) {
            float sum = w;
            for (int o = p.half_k; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (chosen) w = __fdividef(w, sum);
        }
        if (token && my_place < p.top_k) {
            p.weights[t * p.top_k + my_place] = w * p.scale;
            p.experts[t * p.top_k + my_place] = expert;
        }
    };

    constexpr int kUnsure = -2;
    bool any_unsure = false;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kRouteWarps * p.batch;
    for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp) * p.batch; t0 < p.T; t0 += step) {
        const int count = static_cast<int>(min(static_cast<int64_t>(p.batch), p.T - t0));
        uint32_t mine = 0, left = 0;  // of the token of my_slot: the key of my_place, and that of the first expert left out
        int owner = 0;  // the lane that it comes from
        float row_max = 0.0f, denominator = 1.0f;
        bool unsure = false;
        for (int q = 0; q < count; ++q) {
            float c[V];
            route_load_lane<T, V>(static_cast<const T*>(p.logits) + (t0 + q) * p.E, lane * V, p.E, p.vec, c);
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = route_logit(c[i]);
            float m = 0.0f, z = 1.0f;
            if (need_denominator) {
                route_denominator(c, m, z);
                if (my_slot == q) row_max = m, denominator = z;
            }
            auto score = [&](float v) { return softmax ? __fdividef(expf(v - m), z) : approx_reciprocal(1.0f + __expf(-v)); };
            if (by_scores) {
                if (softmax) {
#pragma unroll
                    for (int i = 0; i < V; ++i) c[i] = c[i] > -INFINITY ? fmaxf(__fdividef(expf(c[i] - m), z) + bias[i], -INFINITY) : -INFINITY;
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) c[i] = c[i] > -INFINITY ? fmaxf(approx_reciprocal(1.0f + __expf(-c[i])) + bias[i], -INFINITY) : -INFINITY;
                }
            }
            if (p.groups > 1) {
                float first, second;
                int g;
                if (scores_of_groups) {
                    float of_group[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) of_group[i] = c[i] > -INFINITY ? score(c[i]) : -INFINITY;
                    g = route_group_best(p, of_group, scratch, first, second);
                } else {
                    g = route_group_best(p, c, scratch, first, second);
                }
                const float value = route_group_value(p, first, second);
                // The place of this lane's group in their order; the lowest value kept and the highest one dropped.
                const int span = scratch ? 1 : p.E / p.groups / V;
                int rank = 0;
                for (int o = 0; o < p.groups; ++o) {
                    const float other = __shfl_sync(0xffffffffu, value, o * span);
                    rank += other > value || (other == value && o < g);
                }
                const bool live = g >= 0 && value > -INFINITY, kept = live && rank < p.top_groups;
                if (by_scores || scores_of_groups) {
                    const bool close = route_groups_close(value, route_group_slack<V>(p, first, second, softmax), live, kept);
                    if (my_slot == q) unsure = close;
                }
                if (!scratch) {
#pragma unroll
                    for (int i = 0; i < V; ++i) c[i] = kept ? c[i] : -INFINITY;
                } else {
                    route_drop_groups(p, __ballot_sync(0xffffffffu, kept), g, false, c);
                }
            }
            uint32_t key[V];
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = (route_key(c[i]) & ~kPlace) | (kPlace - i);
            route_sort(key);
            const int at = q * wide;
            for (int j = 0; j < p.top_k; ++j) {
                const uint32_t top = warp_max_key(key[0]);
                if (top <= kRouteNone) break;
                // the first lane that has this value, and the first place there
                const int src = __ffs(__ballot_sync(0xffffffffu, (key[0] | kPlace) == (top | kPlace))) - 1;
                const uint32_t taken = __shfl_sync(0xffffffffu, key[0], src);
                if (lane == at + j) mine = taken, owner = src;
                const bool next = lane == src;
#pragma unroll
                for (int i = 0; i + 1 < V; ++i) key[i] = next ? key[i + 1] : key[i];
                key[V - 1] = next ? 0u : key[V - 1];
            }
            if (!exact) {
                const uint32_t rest = warp_max_key(key[0]);
                if (my_slot == q) left = rest;
            }
        }
        if (!exact) {
            // Neighbours in the order, the first one left out among them; what keys drop below a value is at most their lowest bits' worth of it.
            uint32_t after = __shfl_down_sync(0xffffffffu, mine, 1);
            if (my_place + 1 >= p.top_k) after = left;
            if (my_place < p.top_k && mine > kRouteNone && after > kRouteNone) {
                const float a = route_unkey(mine & ~kPlace), b = route_unkey(after & ~kPlace);
                const float lost = (kPlace + 1) * 1.1920929e-7f * fmaxf(fabsf(a), fabsf(b));
                unsure = unsure || a - b <= (by_scores ? route_margin<V>(a, softmax) + lost : lost);
            }
        }
        int expert = mine > kRouteNone ? owner * V + static_cast<int>(kPlace - (mine & kPlace)) : -1;
        // What fp32 cannot tell is marked, and decided behind the loop.
        const uint32_t again = __ballot_sync(0xffffffffu, unsure);
        if (again >> (my_slot * wide) & (wide == 32 ? 0xffffffffu : (1u << wide) - 1u)) expert = kUnsure;
        any_unsure = any_unsure || again != 0;
        finish(t0 + my_slot, my_slot < count, expert, row_max, denominator);
    }
    if (!any_unsure) return;
    __syncwarp();
    for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp) * p.batch; t0 < p.T; t0 += step) {
        const int count = static_cast<int>(min(static_cast<int64_t>(p.batch), p.T - t0));
        const int32_t mark = lane < count ? *reinterpret_cast<const volatile int32_t*>(p.experts + (t0 + lane) * p.top_k) : 0;
        for (uint32_t again = __ballot_sync(0xffffffffu, mark == kUnsure); again; again &= again - 1) {
            const int64_t t = t0 + __ffs(again) - 1;
            float m, z;
            const int expert = route_carefully<T, V>(p, static_cast<const T*>(p.logits) + t * p.E, exact_c, use_scratch, m, z);
            finish(t, my_slot == 0, expert, m, z);
        }
    }
}

}  // namespace gi8
