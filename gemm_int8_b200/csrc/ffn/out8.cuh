// What the operators around the products share: eight values a lane in, 8-bit values and their scale out.
//   int8   s = amax / 127,  q = clamp(rint(v / s), -127, 127)
//   e4m3   s = amax / 448,  q = v / s rounded to e4m3 (half to even)
// with s = 1 where all values are zero, or so small that s would be.  A NaN or infinity among the values makes the scale NaN or infinite, so that every product with
// them shows it (an int8 has no value of its own for it).
#pragma once

#include "../k_quant.cuh"

namespace gi8 {

enum class Out8 { kInt8, kE4m3 };

// Maximum of magnitudes that propagates NaN.
GI8_DEVICE float amax8_nan(const uint64_t (&v)[4])
{
    float a, b, c, d, e, f, g, h;
    f32x2_split(v[0], a, b), f32x2_split(v[1], c, d), f32x2_split(v[2], e, f), f32x2_split(v[3], g, h);
    return max3_abs_nan(max3_abs_nan(a, b, c), max3_abs_nan(d, e, f), max3_abs_nan(g, h, 0.0f));
}

GI8_DEVICE float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

GI8_DEVICE float warp_max_nan(float m)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// r: an approximate (int8) or the nearest (e4m3) reciprocal of s; NaN where the quick forms below do not hold.
template <Out8 OUT>
GI8_DEVICE QuantScale make_out_scale(float amax)
{
    QuantScale q;
    q.s = __fdiv_rn(amax, OUT == Out8::kInt8 ? 127.0f : 448.0f);
    if (q.s == 0.0f) q.s = 1.0f;
    if constexpr (OUT == Out8::kInt8) asm("rcp.approx.f32 %0, %1;" : "=f"(q.r) : "f"(q.s));
    else q.r = __frcp_rn(q.s);
    if (!(q.s > (OUT == Out8::kInt8 ? 1e-30f : 1e-20f) && q.s < 1e30f)) q.r = __int_as_float(0x7fffffff);
    return q;
}

// Scales of U values a lane over runs of sixteen lanes (128-wide blocks), one division a lane instead of U: while a butterfly doubles the lanes
// that a value has been reduced over it halves the values that a lane is in charge of, so that in the end each lane holds the maximum of one of them,
// makes its scale, and fetches the others'.  (As group_scales of k_quant.cuh, for either type, and with NaN.)
template <Out8 OUT, int U>
GI8_DEVICE void block_scales(float (&m)[U], QuantScale (&qs)[U])
{
    static_assert(U == 1 || U == 2 || U == 4 || U == 8, "values a lane");
    const int lane = threadIdx.x & 31;
    int n = U;
#pragma unroll
    for (int o = 1; o < U; o <<= 1) {
        n >>= 1;
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < U / 2; ++i) {
            if (i < n) {
                const float keep = up ? m[i + n] : m[i], give = up ? m[i] : m[i + n];
                m[i] = max_nan(keep, __shfl_xor_sync(0xffffffffu, give, o));
            }
        }
    }
#pragma unroll
    for (int o = U; o < 16; o <<= 1) m[0] = max_nan(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
    const QuantScale mine = make_out_scale<OUT>(m[0]);
    const int first = lane & ~15;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        // the lane whose lowest bits are those of u from the highest down
        int src = first;
#pragma unroll
        for (int b = 1, h = U / 2; b < U; b <<= 1, h >>= 1) src += u & h ? b : 0;
        qs[u].s = U == 1 ? mine.s : __shfl_sync(0xffffffffu, mine.s, src);
        qs[u].r = U == 1 ? mine.r : __shfl_sync(0xffffffffu, mine.r, src);
    }
}

// Two floats -> two packed e4m3 (lo in the low byte).
GI8_DEVICE uint32_t cvt_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Four values -> four packed e4m3 of v / s, the quotient as IEEE division gives it: from the nearest reciprocal r and t = v r the exact
// remainder v - t s corrects t (P. Markstein, IBM J. Res. Dev. 34, 1990), two multiply-adds on packed pairs; a quotient that lies
// between two e4m3 numbers comes out exactly there.  Scales from 1e-20 on keep the remainder of every quotient that does not round to
// zero in range; the others (r is NaN) take the division itself.
// What is computed is -v / s, whose sign bits one XOR turns round: from v = -0 the sums above would give +0, as (-0)(-s) - 0 = +0; from t = +0 they keep the
// sign that division gives.
GI8_DEVICE uint32_t e4m3_pack4(uint64_t v0, uint64_t v1, const QuantScale& qs)
{
    const uint64_t nr2 = f32x2(-qs.r, -qs.r), s2 = f32x2(qs.s, qs.s);
    const uint64_t t0 = mul2(v0, nr2), t1 = mul2(v1, nr2);
    float a, b, c, d;
    f32x2_split(fma2(fma2(t0, s2, v0), nr2, t0), a, b), f32x2_split(fma2(fma2(t1, s2, v1), nr2, t1), c, d);
    return (cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16)) ^ 0x80808080u;
}

GI8_DEVICE uint32_t e4m3_pack4_exact(uint64_t v0, uint64_t v1, float s)
{
    float a, b, c, d;
    f32x2_split(v0, a, b), f32x2_split(v1, c, d);
    return cvt_e4m3x2(__fdiv_rn(a, s), __fdiv_rn(b, s)) | (cvt_e4m3x2(__fdiv_rn(c, s), __fdiv_rn(d, s)) << 16);
}

// LOADS x eight values with the scale of each (or one for all) -> put(u, eight bytes).  Called by whole warps, which look once whether any scale of
// theirs is out of the quick form's range (SwiGLU of 4096 x 14336 49.3 -> 48.0 us against a look at every four values).
template <Out8 OUT, int LOADS, int SCALES, typename Put>
GI8_DEVICE void out8_store(const uint64_t (&v)[LOADS][4], const QuantScale (&qs)[SCALES], Put put)
{
    static_assert(SCALES == LOADS || SCALES == 1, "a scale for each eight values, or one");
    if constexpr (OUT == Out8::kInt8) {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const QuantScale& q = qs[SCALES == 1 ? 0 : u];
            put(u, make_uint2(quant_pack4(v[u][0], v[u][1], q), quant_pack4(v[u][2], v[u][3], q)));
        }
    } else {
        bool quick = true;
#pragma unroll
        for (int u = 0; u < SCALES; ++u) quick = quick && qs[u].r == qs[u].r;
        if (__all_sync(0xffffffffu, quick)) {
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const QuantScale& q = qs[SCALES == 1 ? 0 : u];
                put(u, make_uint2(e4m3_pack4(v[u][0], v[u][1], q), e4m3_pack4(v[u][2], v[u][3], q)));
            }
        } else {
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const float s = qs[SCALES == 1 ? 0 : u].s;
                put(u, make_uint2(e4m3_pack4_exact(v[u][0], v[u][1], s), e4m3_pack4_exact(v[u][2], v[u][3], s)));
            }
        }
    }
}

// Eight consecutive values as they lie in memory (16 or 32 bytes, aligned to 16), and as fp32 pairs.
template <typename T>
struct Raw8 {
    uint4 u[sizeof(T) / 2];
};

template <typename T>
GI8_DEVICE Raw8<T> load8(const T* p)
{
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.u[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}

template <typename T>
GI8_DEVICE Raw8<T> zero8()
{
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.u[i] = make_uint4(0u, 0u, 0u, 0u);
    return r;
}

template <typename T>
GI8_DEVICE void unpack8(const Raw8<T>& r, uint64_t (&v)[4])
{
    if constexpr (sizeof(T) == 2) {
        unpack16<T>(r.u[0], v);
    } else {
        unpack16<T>(r.u[0], reinterpret_cast<uint64_t(&)[2]>(v[0]));
        unpack16<T>(r.u[1], reinterpret_cast<uint64_t(&)[2]>(v[2]));
    }
}

// Eight fp32 values -> memory, rounded to T.
template <typename T>
GI8_DEVICE void store8(T* p, const uint64_t (&v)[4])
{
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) f32x2_split(v[i], f[2 * i], f[2 * i + 1]);
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    } else {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
}

}  // namespace gi8
