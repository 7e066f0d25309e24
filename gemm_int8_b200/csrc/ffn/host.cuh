// C ABI of the operators around the products of a feed-forward block.  Included at the end of api.cu, whose helpers it uses.
#pragma once

#include "k_act.cuh"
#include "k_norm.cuh"

namespace {

constexpr int64_t kMaxNormFeatures = kNormThreads * 64;  // 64 values a thread

int check_out8(const void* q, int q_type, const float* scales, int block_scales, int64_t M, int64_t K)
{
    if (M < 0 || K < 0) return fail(GI8_ERR_INVALID_ARGUMENT, "negative dimension");
    if (q_type != 0 && q_type != 1) return fail(GI8_ERR_INVALID_ARGUMENT, "q_type must be 0 (int8) or 1 (e4m3)");
    if (q_type == 1 && !block_scales) return fail(GI8_ERR_INVALID_ARGUMENT, "e4m3 has a scale per 128 columns, which its product takes");
    if (K % 16) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld features: they must be a multiple of 16", (long long)K);
    if (M > INT32_MAX) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "M must be below 2^31");
    if (K >= kMaxK) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld features: there must be fewer than %lld", (long long)K, (long long)kMaxK);
    if (M == 0 || K == 0) return GI8_OK;
    if (!q || !scales) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(q, 8) || misaligned(scales, 4)) return fail(GI8_ERR_MISALIGNED, "q must be 8-byte and scales 4-byte aligned");
    return GI8_OK;
}

// Values a thread: 32, which wants the fewest warps a row and the most rows on an SM (16384 x 8192 bf16 with a residual, 8 / 16 / 32 / 64 values: 179 / 176 /
// 141 / 163 us; 16384 x 4096 without one 71 / 64 / 54, and 50 since 32 values have at most 64 registers); 16 where there is no second row for an SM to work on beside (148 x 8192: 4.5 us for 6.3; level from
// 592 rows on), 64 where 512 threads of 32 would not hold the row.
template <typename TX, typename TR, typename TW, Out8 OUT, bool BLOCK>
int launch_norm(NormParams p, int sms, cudaStream_t s)
{
    const int vectors = (p.H + 7) / 8;
    // (two loads a thread: two warps for each of the form of four, whose order of summing up they keep; rows that one warp of that form holds stay with it)
    auto go = [&](auto kernel, int loads) {
        p.row_warps = loads == 2 ? (vectors + 127) / 128 * 2 : (vectors + 32 * loads - 1) / (32 * loads);
        const int rows = p.row_warps == 1 ? 8 : 1;
        return launch(kernel, dim3(static_cast<unsigned>((p.M + rows - 1) / rows)), p.row_warps * rows * 32, 0, s, dim3(1), knobs().pdl, p);
    };
    if (p.M <= 2 * sms && vectors > 128 && vectors <= 2 * kNormThreads) return go(rms_norm_quantize_kernel<TX, TR, TW, OUT, BLOCK, 2>, 2);
    if (vectors <= 4 * kNormThreads) return go(rms_norm_quantize_kernel<TX, TR, TW, OUT, BLOCK, 4>, 4);
    return go(rms_norm_quantize_kernel<TX, TR, TW, OUT, BLOCK, 8>, 8);
}

template <typename TX, typename TR, typename TW>
int launch_norm(const NormParams& p, int q_type, int block_scales, int sms, cudaStream_t s)
{
    if (q_type == 1) return launch_norm<TX, TR, TW, Out8::kE4m3, true>(p, sms, s);
    if (block_scales) return launch_norm<TX, TR, TW, Out8::kInt8, true>(p, sms, s);
    return launch_norm<TX, TR, TW, Out8::kInt8, false>(p, sms, s);
}

template <typename TX, typename TR>
int launch_norm(const NormParams& p, int weight_dtype, int q_type, int block_scales, int sms, cudaStream_t s)
{
    return weight_dtype == 0 ? launch_norm<TX, TR, float>(p, q_type, block_scales, sms, s) : launch_norm<TX, TR, __nv_bfloat16>(p, q_type, block_scales, sms, s);
}

template <typename TX>
int launch_norm(const NormParams& p, int residual_dtype, int weight_dtype, int q_type, int block_scales, int sms, cudaStream_t s)
{
    if (!p.residual) return launch_norm<TX, void>(p, weight_dtype, q_type, block_scales, sms, s);
    return residual_dtype == 0 ? launch_norm<TX, float>(p, weight_dtype, q_type, block_scales, sms, s) : launch_norm<TX, __nv_bfloat16>(p, weight_dtype, q_type, block_scales, sms, s);
}

// Block scales: 32 values a lane, of the two fp32 halves 16, each item on a warp of its own (4096 x 14336 bf16 SwiGLU with 8 / 16 / 32 values 66 / 58 / 49 us;
// a grid of as many CTAs as are resident, whose warps take item after item, 53; e4m3 quantiser of 16384 x 8192 fp32 98, resident CTAs 104).
template <typename T, bool SWIGLU, Out8 OUT>
int launch_act_block(const ActParams& p, cudaStream_t s)
{
    constexpr int LOADS = SWIGLU && sizeof(T) == 4 ? 2 : 4;
    const int64_t items = p.M * ((p.KB + 2 * LOADS - 1) / (2 * LOADS));
    if (items >= (int64_t(1) << 31)) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "too many quantisation blocks");
    return launch(act_quantize_block_kernel<T, SWIGLU, OUT, LOADS>, dim3(static_cast<unsigned>((items + kActThreads / 32 - 1) / (kActThreads / 32))), kActThreads, 0, s,
                  dim3(1), knobs().pdl, p);
}

// A scale per row: 32 values a thread (4096 x 14336 bf16 with 16 / 32 / 64 values 79 / 62 / 78 us, 8192 x 4096 39 / 35 / 57).
template <typename T>
int launch_swiglu_row(const ActParams& p, int sms, cudaStream_t s)
{
    constexpr int LOADS = 4;
    const int vectors = (p.K + 7) / 8;
    const int threads = std::min(1024, (vectors + 32 * LOADS - 1) / (32 * LOADS) * 32);
    return launch(swiglu_quantize_row_kernel<T, LOADS>, dim3(static_cast<unsigned>(std::min<int64_t>(p.M, static_cast<int64_t>(sms) * 8))), threads, 0, s, dim3(1),
                  knobs().pdl, p);
}

}  // namespace

extern "C" {

int gi8_rms_norm_quantize(const void* x, int x_dtype, const void* residual, int residual_dtype, const void* weight, int weight_dtype, float eps, void* total,
                          void* q, int q_type, float* scales, int block_scales, int64_t M, int64_t H, void* stream)
{
    for (int d : {x_dtype, residual_dtype, weight_dtype})
        if (d != 0 && d != 1) return fail(GI8_ERR_INVALID_ARGUMENT, "dtypes must be 0 (fp32) or 1 (bf16)");
    if (int rc = check_out8(q, q_type, scales, block_scales, M, H)) return rc;
    if (H > kMaxNormFeatures) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld features: a norm is over at most %lld", (long long)H, (long long)kMaxNormFeatures);
    // (squares below fp32's range are nothing next to such an eps)
    if (!(eps >= 1e-20f && eps <= 1e20f)) return fail(GI8_ERR_INVALID_ARGUMENT, "eps must lie between 1e-20 and 1e20");
    if (M == 0 || H == 0) return GI8_OK;
    if (!x || !weight || (residual && !total)) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(x, 16) || misaligned(residual, 16) || misaligned(weight, 16) || (residual && misaligned(total, 16)))
        return fail(GI8_ERR_MISALIGNED, "x, residual, weight and total must be 16-byte aligned");
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    NormParams p{};
    p.x = x, p.residual = residual, p.weight = weight, p.total = total, p.q = static_cast<uint8_t*>(q), p.s = scales, p.M = M, p.H = static_cast<int>(H);
    p.KB = static_cast<int>((H + 127) / 128), p.eps = eps, p.inv_h = 1.0f / static_cast<float>(H);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int sms = st->sm_count;
    return x_dtype == 0 ? launch_norm<float>(p, residual_dtype, weight_dtype, q_type, block_scales, sms, s)
                        : launch_norm<__nv_bfloat16>(p, residual_dtype, weight_dtype, q_type, block_scales, sms, s);
}

int gi8_swiglu_quantize(const void* gate_up, int dtype, void* q, int q_type, float* scales, int block_scales, int64_t M, int64_t N, void* stream)
{
    if (dtype != 0 && dtype != 1) return fail(GI8_ERR_INVALID_ARGUMENT, "dtype must be 0 (fp32) or 1 (bf16)");
    if (int rc = check_out8(q, q_type, scales, block_scales, M, N)) return rc;
    if (M == 0 || N == 0) return GI8_OK;
    if (!gate_up) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(gate_up, 16)) return fail(GI8_ERR_MISALIGNED, "gate_up must be 16-byte aligned");
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    ActParams p{gate_up, static_cast<uint8_t*>(q), scales, M, static_cast<int>(N), static_cast<int>((N + 127) / 128)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int sms = st->sm_count;
    if (!block_scales) return dtype == 0 ? launch_swiglu_row<float>(p, sms, s) : launch_swiglu_row<__nv_bfloat16>(p, sms, s);
    if (q_type == 1)
        return dtype == 0 ? launch_act_block<float, true, Out8::kE4m3>(p, s) : launch_act_block<__nv_bfloat16, true, Out8::kE4m3>(p, s);
    return dtype == 0 ? launch_act_block<float, true, Out8::kInt8>(p, s) : launch_act_block<__nv_bfloat16, true, Out8::kInt8>(p, s);
}

}  // extern "C"
