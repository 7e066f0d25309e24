// C ABI of the experts' operators: argument checks, the choice of a tile, launches.  Included at the end of api.cu, whose helpers it
// uses.
#pragma once

#include "k_combine.cuh"
#include "k_experts_gemm.cuh"
#include "k_group.cuh"
#include "k_route.cuh"

namespace {

// Kernels whose shared-memory limit has been raised, a bit each (DeviceState::attr_set is full).
std::atomic<uint64_t> g_experts_attr[kMaxDevices];

template <typename Kernel>
int experts_smem(int slot, Kernel kernel, size_t bytes)
{
    int dev = 0;
    GI8_CUDA(cudaGetDevice(&dev));
    if (!((g_experts_attr[dev].load() >> slot) & 1)) {
        GI8_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
        g_experts_attr[dev].fetch_or(uint64_t(1) << slot);
    }
    return GI8_OK;
}

bool misaligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

template <typename T, int V>
int launch_route(RouteParams p, int sms, cudaStream_t s)
{
    // Groups that are not whole runs of a power of two of lanes have their values looked up through shared memory.
    int use_scratch = 0;
    if (p.groups > 1) {
        const int size = p.E / p.groups, span = size / V;
        use_scratch = size % V != 0 || (span & (span - 1)) != 0;
    }
    const size_t smem = static_cast<size_t>(kRouteWarps) * p.E * sizeof(double);
    // As many CTAs as are resident: a warp takes batch after batch of its tokens.
    const int64_t resident = static_cast<int64_t>(sms) * (V <= 8 ? 8 : 3);
    p.batch = static_cast<int>(std::min<int64_t>(32 / (p.half_k > 0 ? 2 * p.half_k : 1), std::max<int64_t>(1, p.T / (resident * kRouteWarps))));
    const int64_t per_cta = static_cast<int64_t>(kRouteWarps) * p.batch;
    const int64_t ctas = std::min<int64_t>((p.T + per_cta - 1) / per_cta, resident);
    return launch(route_experts_kernel<T, V>, dim3((unsigned)ctas), kRouteWarps * 32, smem, s, dim3(1), knobs().pdl, p, use_scratch);
}

template <typename T>
int launch_route_for(RouteParams p, int sms, cudaStream_t s)
{
    const int per_lane = (p.E + 31) / 32;
    auto vec = [&](const void* base, int v, int size) { return p.E % v == 0 && !misaligned(base, 16) && v * size % 16 == 0; };
    for (p.half_k = 1; 2 * p.half_k < p.top_k;) p.half_k *= 2;
    if (p.top_k == 1) p.half_k = 0;
#define GI8_ROUTE(V_)                                              \
    if (per_lane <= V_) {                                          \
        p.vec = vec(p.logits, V_, static_cast<int>(sizeof(T)));    \
        p.vec_bias = vec(p.bias, V_, 4);                           \
        return launch_route<T, V_>(p, sms, s);                     \
    }
    GI8_ROUTE(1)
    GI8_ROUTE(2)
    GI8_ROUTE(4)
    GI8_ROUTE(5)  // 129 to 160 experts (160 with groups, bias: 4096 tokens 8.8 us, eight to a lane 15.0; 16 tokens 3.4 and 4.2)
    GI8_ROUTE(8)
    GI8_ROUTE(16)
    GI8_ROUTE(32)
#undef GI8_ROUTE
    return fail(GI8_ERR_UNSUPPORTED_SHAPE, "too many experts");
}

// Gate and up rows of int8 weights [E, 2, N, K] in alternating runs of 16 (N a multiple of 16): dimensions K, row of a run, half, run, expert.
// A box of 128 bytes x 16 x 2 x 4 x 1 is the weight tile of 64 channels.
int make_gate_up_map(CUtensorMap* map, const int8_t* w, int64_t E, int64_t N, int64_t K)
{
    return cached_map(map, MapKey{w, static_cast<uint64_t>(K), static_cast<uint64_t>(N), static_cast<uint64_t>(E), 0u, 0u, 3u});
}

template <int WARPS, int LOADS, GroupStep STEP>
int launch_group(GroupParams p, int ctas, int slot, cudaStream_t s)
{
    auto kernel = group_by_expert_kernel<WARPS, LOADS, STEP>;
    auto smem = [](int64_t E) { return static_cast<size_t>((WARPS + 3) * E + WARPS * 32 * LOADS) * 4; };
    static_assert((WARPS + 3) * kGroupMaxExperts * 4 + WARPS * 32 * LOADS * 4 <= 227 * 1024 - 1024, "fits shared memory at the most experts");
    if (int rc = experts_smem(slot, kernel, smem(kGroupMaxExperts))) return rc;
    p.per_warp = static_cast<int>((p.S + static_cast<int64_t>(ctas) * WARPS * 32 - 1) / (ctas * WARPS * 32)) * 32;
    return launch(kernel, dim3(ctas), WARPS * 32, smem(p.E), s, dim3(1), knobs().pdl, p);
}

// CTAs of a grouping: 1 up to 8192 pairs; of 2048 pairs up to 262144, of 16384 above.
constexpr int64_t kGroupMaxPairs = int64_t(1) << 24;
int group_ctas(int64_t S) { return S <= 8192 ? 1 : static_cast<int>(S <= 262144 ? (S + 2047) / 2048 : (S + 16383) / 16384); }

template <int BT, int STAGES, bool SWIGLU, bool PAIR, bool GATHER>
int launch_experts(DeviceState* st, int slot, const int8_t* w, ExpertsParams p, cudaStream_t s)
{
    constexpr int kRowsX = PAIR ? BT / 2 : BT;
    constexpr size_t smem = static_cast<size_t>(STAGES) * (kBM + kRowsX) * kBK + experts_turn_bytes(SWIGLU, PAIR) + 1024;
    auto kernel = experts_gemm_kernel<BT, STAGES, SWIGLU, PAIR, GATHER>;
    if (int rc = experts_smem(slot, kernel, smem)) return rc;
    CUtensorMap mw;
    TokenMaps mx;
    const int64_t rows_w = static_cast<int64_t>(p.E) * p.N * (SWIGLU ? 2 : 1);
    p.interleave = SWIGLU && p.N % 16 == 0;
    if (p.interleave) {
        if (int rc = make_gate_up_map(&mw, w, p.E, p.N, p.K)) return rc;
    } else if (int rc = make_operand_map(&mw, w, rows_w, p.K, SWIGLU ? 16 : kBM)) {
        return rc;
    }
    for (int i = 0; i < 4; ++i) {
        if (GATHER) mx.m[i] = mw;  // (unused by the kernel)
        else if (int rc = make_operand_map(&mx.m[i], p.x, p.tokens, p.K, (i + 1) * kRowsX / 4)) return rc;
    }
    // A band's rows take about 16 MB, as in the dense kernel (one expert, 32768 rows, 4096 x 4096, for a second on end, without bands and with: 547 and 430 us).
    p.band = static_cast<int>(std::min<int64_t>(64, std::max<int64_t>(4, (int64_t(16) << 20) / (static_cast<int64_t>(BT) * p.K))));
    const int channels = (SWIGLU ? kBM / 2 : kBM) * (PAIR ? 2 : 1);
    const int64_t token_tiles = std::min<int64_t>(p.rows, p.E + p.rows / BT);  // at most
    const int64_t tiles = token_tiles * ((p.N + channels - 1) / channels);
    const int64_t slots = BT == 64 ? 2 * st->sm_count : PAIR ? st->sm_count / 2 : st->sm_count;
    const int grid = static_cast<int>(std::min<int64_t>(tiles, slots)) * (PAIR ? 2 : 1);
    return launch(kernel, dim3(grid), experts_threads(GATHER), smem, s, dim3(PAIR ? 2 : 1), knobs().pdl, mw, mx, p);
}

// The form of a product, by the rows that an expert can be expected to have (half as many again as on average, or all that it can have
// if no token names it twice):
//   up to 64   one-CTA tiles of 64 tokens, two CTAs per SM, so that the next launch's CTAs can sit down beside this one's; where the tiles
//              leave SMs without one for long, tiles of 32 tokens with ten stages, more bytes in flight for the few
//   more       two-CTA tiles of 256 tokens
// us (graph replays), tiles of 64 / 256 tokens, at 32, 40, 48, 64 and 128 rows per expert on average (the rule changes over at 43):
//   E = 64, k = 8, product 4096 x 1408, rows in order  59.4 / 57.0   63.6 / 63.2   64.6 / 63.6   67.3 / 65.4   94.4 / 74.1
//                                       gathered       61.7 / 61.4   64.7 / 64.9   67.4 / 65.3   68.9 / 67.7   99.2 / 76.6
//   SwiGLU 1408 x 4096, rows in order                   110 / 115     121 / 122     118 / 125     127 / 126     194 / 136
//                       gathered                        112 / 120     120 / 123     120 / 123     128 / 126     207 / 140
//   E = 8, k = 2, product 4096 x 14336, rows in order  73.8 / 78.7   75.9 / 81.0   97.3 / 80.8   95.5 / 82.0
// One limit for all of them is within 6 % of the better form here.  (One-CTA tiles of 128 tokens were level with or behind the better of the
// two everywhere.)  One token to two experts, product 4096 x 14336, 64 tiles: 40.0, ten stages 32.0 (one to six, 2048 x 1408, 96 short
// tiles: 8.3 and 9.7).
enum ExpertsForm { EXPERTS_FEW, EXPERTS_64, EXPERTS_256 };

ExpertsForm experts_form(const ExpertsParams& p, bool swiglu, int sms)
{
    const int64_t most = p.slots ? p.tokens : p.rows;
    const int64_t want = std::min(most, (3 * p.rows / 2 + p.E - 1) / p.E);
    if (want > 64) return EXPERTS_256;
    const int channels = swiglu ? kBM / 2 : kBM;
    const int64_t tiles = std::min<int64_t>(p.rows, p.E + p.rows / 32) * ((p.N + channels - 1) / channels);
    return want <= 32 && tiles <= sms && p.K >= 48 * kBK ? EXPERTS_FEW : EXPERTS_64;
}

template <bool SWIGLU, bool GATHER>
int dispatch_experts(DeviceState* st, const int8_t* w, const ExpertsParams& p, cudaStream_t s)
{
    constexpr int slot = (SWIGLU ? 4 : 0) + (GATHER ? 16 : 0);
    switch (experts_form(p, SWIGLU, st->sm_count)) {
        case EXPERTS_FEW: return launch_experts<32, 10, SWIGLU, false, GATHER>(st, slot, w, p, s);
        case EXPERTS_64: return launch_experts<64, 4, SWIGLU, false, GATHER>(st, slot + 1, w, p, s);
        default: return launch_experts<256, 6, SWIGLU, true, GATHER>(st, slot + 2, w, p, s);
    }
}

}  // namespace

extern "C" {

int gi8_route_experts(const void* logits, int logits_dtype, const float* bias, float* weights, int32_t* experts, int64_t T, int64_t E,
                      int64_t top_k, int sigmoid, int64_t groups, int64_t top_groups, int group_top2, int renormalize, float scale,
                      void* stream)
{
    if (T < 0 || T > INT32_MAX) return fail(GI8_ERR_INVALID_ARGUMENT, "T=%lld must be in [0, 2^31)", (long long)T);
    if (logits_dtype != 0 && logits_dtype != 1) return fail(GI8_ERR_INVALID_ARGUMENT, "logits_dtype must be 0 (fp32) or 1 (bf16)");
    if (E < 1 || E > kRouteMaxExperts) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld experts: 1 to %d are supported", (long long)E, kRouteMaxExperts);
    if (top_k < 1 || top_k > kRouteMaxTopK || top_k > E)
        return fail(GI8_ERR_UNSUPPORTED_SHAPE, "top_k=%lld must be in [1, min(%d, experts)]", (long long)top_k, kRouteMaxTopK);
    if (groups < 1 || groups > kRouteMaxGroups || E % groups)
        return fail(GI8_ERR_UNSUPPORTED_SHAPE, "groups=%lld must divide the %lld experts and be at most %d", (long long)groups, (long long)E, kRouteMaxGroups);
    if (top_groups < 1 || top_groups > groups || top_k > top_groups * (E / groups))
        return fail(GI8_ERR_UNSUPPORTED_SHAPE, "top_groups=%lld must be in [1, groups] and hold top_k experts", (long long)top_groups);
    if (T == 0) return GI8_OK;
    if (!logits || !weights || !experts) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(logits, logits_dtype == 0 ? 4 : 2) || misaligned(bias, 4) || misaligned(weights, 4) || misaligned(experts, 4))
        return fail(GI8_ERR_MISALIGNED, "a pointer is not aligned to its elements");
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    RouteParams p{};
    p.logits = logits, p.bias = bias, p.weights = weights, p.experts = experts;
    p.T = (int)T, p.E = (int)E, p.top_k = (int)top_k, p.sigmoid = sigmoid != 0;
    p.groups = top_groups == groups ? 1 : (int)groups, p.top_groups = (int)top_groups;  // where all groups are kept there are none
    p.group_top2 = group_top2 != 0, p.renormalize = renormalize != 0, p.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return logits_dtype == 0 ? launch_route_for<float>(p, st->sm_count, s) : launch_route_for<__nv_bfloat16>(p, st->sm_count, s);
}

int64_t gi8_group_by_expert_workspace_bytes(int64_t S, int64_t E)
{
    if (S <= 0 || S > kGroupMaxPairs || E <= 0 || E > kGroupMaxExperts) return 0;
    const int ctas = group_ctas(S);
    return ctas > 1 ? 4 * E * ctas : 0;
}

int gi8_group_by_expert(const int32_t* experts, int64_t S, int64_t E, int64_t first, int32_t* offsets, int32_t* slots, int32_t* places, void* workspace,
                        int64_t workspace_bytes, void* stream)
{
    if (S < 0 || S > kGroupMaxPairs) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "S=%lld must be in [0, 2^24]", (long long)S);
    if (E < 1 || E > kGroupMaxExperts) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld experts: 1 to %d are supported", (long long)E, kGroupMaxExperts);
    if (first < 0 || first > INT32_MAX - E) return fail(GI8_ERR_INVALID_ARGUMENT, "first expert %lld out of range", (long long)first);
    if (!offsets || (S > 0 && (!experts || !slots || !places))) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(experts, 4) || misaligned(offsets, 4) || misaligned(slots, 4) || misaligned(places, 4))
        return fail(GI8_ERR_MISALIGNED, "a pointer is not 4-byte aligned");
    const int64_t needed = gi8_group_by_expert_workspace_bytes(S, E);
    if (needed > 0 && (!workspace || workspace_bytes < needed))
        return fail(GI8_ERR_WORKSPACE, "grouping %lld pairs needs %lld bytes of workspace, got %lld", (long long)S, (long long)needed, (long long)workspace_bytes);
    if (misaligned(workspace, 4)) return fail(GI8_ERR_MISALIGNED, "workspace must be 4-byte aligned");
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    GroupParams p{};
    p.experts = experts, p.offsets = offsets, p.slots = slots, p.places = places;
    p.S = (int)S, p.E = (int)E, p.first = (int)first;
    while ((E >> p.bits) != 0) ++p.bits;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.counts = static_cast<int32_t*>(workspace);
    const int ctas = group_ctas(S);
    if (S <= 2048) return launch_group<8, 8, GROUP_ALL>(p, 1, 8, s);
    if (S <= 8192) return launch_group<32, 8, GROUP_ALL>(p, 1, 9, s);
    if (S <= 262144) {
        if (int rc = launch_group<16, 4, GROUP_COUNT>(p, ctas, 10, s)) return rc;
        return launch_group<16, 4, GROUP_PLACE>(p, ctas, 11, s);
    }
    if (int rc = launch_group<32, 16, GROUP_COUNT>(p, ctas, 12, s)) return rc;
    return launch_group<32, 16, GROUP_PLACE>(p, ctas, 13, s);
}

// early: the launch in front writes neither w nor offsets, and what does had ended when it let this one start (the quantiser of a layer).
static int matmul_experts(const int8_t* x, const int8_t* w, const float* sx, const float* sw, const int32_t* offsets, const int32_t* slots,
                          int64_t top_k, void* out, int64_t rows, int64_t tokens, int64_t E, int64_t N, int64_t K, int swiglu, void* stream,
                          bool early)
{
    if (E < 1 || E > kExpertsMaxExperts) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld experts: 1 to %d are supported", (long long)E, kExpertsMaxExperts);
    if (rows < 0 || tokens < 0 || N < 0) return fail(GI8_ERR_INVALID_ARGUMENT, "negative dimension");
    if (top_k < 1 || top_k > INT32_MAX) return fail(GI8_ERR_INVALID_ARGUMENT, "top_k=%lld must be positive", (long long)top_k);
    if (!slots && tokens < rows) return fail(GI8_ERR_INVALID_ARGUMENT, "%lld rows of x for %lld rows of the result", (long long)tokens, (long long)rows);
    if (tokens > INT32_MAX - 256 || rows > INT32_MAX - 256) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "rows must be below 2^31 - 256");
    // Offsets that do not ascend may give every expert all rows.  The kernel counts token tiles in 32 bits, of 64 rows at least where there are many.
    if (E * ((rows + 63) / 64) > INT32_MAX)
        return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld experts times %lld rows must be below 2^37", (long long)E, (long long)rows);
    if (N > (int64_t(1) << 30) || E * N * (swiglu ? 2 : 1) > INT32_MAX - 256)
        return fail(GI8_ERR_UNSUPPORTED_SHAPE, "%lld experts of %lld channels: together below 2^31 - 256", (long long)E, (long long)N);
    if (int rc = check_common(x, w, out, rows, N, K, 2)) return rc;
    if (rows == 0 || N == 0) return GI8_OK;
    DeviceState* st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (K == 0 || tokens == 0) {
        if (int rc = get_device_state(&st)) return rc;
        return zero_output(out, rows * N * 2, s);
    }
    if (int rc = check_scale_pointers(sx, sw)) return rc;
    if (!offsets) return fail(GI8_ERR_INVALID_ARGUMENT, "null offsets");
    if (misaligned(offsets, 4) || misaligned(slots, 4)) return fail(GI8_ERR_MISALIGNED, "offsets and slots must be 4-byte aligned");
    if (int rc = get_device_state(&st)) return rc;
    ExpertsParams p{};
    p.x = x, p.out = static_cast<uint16_t*>(out), p.sx = sx, p.sw = sw, p.offsets = offsets, p.slots = slots, p.status = st->status;
    p.rows = rows, p.tokens = (int)tokens, p.E = (int)E, p.N = (int)N, p.K = (int)K, p.top_k = (int)top_k;
    p.vec = !misaligned(out, 16) && N % 8 == 0;
    p.weight_policy_first = rows <= 32 * E;
    p.early = early && knobs().pdl;
    if (slots) return swiglu ? dispatch_experts<true, true>(st, w, p, s) : dispatch_experts<false, true>(st, w, p, s);
    return swiglu ? dispatch_experts<true, false>(st, w, p, s) : dispatch_experts<false, false>(st, w, p, s);
}

int gi8_matmul_experts(const int8_t* x, const int8_t* w, const float* sx, const float* sw, const int32_t* offsets, const int32_t* slots,
                       int64_t top_k, void* out, int64_t rows, int64_t tokens, int64_t E, int64_t N, int64_t K, int swiglu, void* stream)
{
    return matmul_experts(x, w, sx, sw, offsets, slots, top_k, out, rows, tokens, E, N, K, swiglu, stream, false);
}

static int combine_experts(const void* y, const float* weights, const int32_t* places, const void* add, bool add_f32, void* out, int64_t T, int64_t top_k,
                           int64_t rows, int64_t N, void* stream)
{
    if (T < 0 || T > INT32_MAX || rows < 0 || rows > INT32_MAX || N < 0 || N > INT32_MAX - 4096) return fail(GI8_ERR_INVALID_ARGUMENT, "a dimension is out of range");
    if (top_k < 1 || top_k > kCombineMaxTopK) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "top_k=%lld must be in [1, %d]", (long long)top_k, kCombineMaxTopK);
    if (T == 0 || N == 0) return GI8_OK;
    if ((!y && rows > 0) || !weights || !places || !out) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(y, 2) || misaligned(add, add_f32 ? 4 : 2) || misaligned(out, 2) || misaligned(weights, 4) || misaligned(places, 4))
        return fail(GI8_ERR_MISALIGNED, "a pointer is not aligned to its elements");
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    CombineParams p{};
    p.y = static_cast<const uint16_t*>(y), p.weights = weights, p.places = places, p.add = add, p.out = static_cast<uint16_t*>(out);
    p.rows = rows, p.T = (int)T, p.N = (int)N, p.top_k = (int)top_k;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool vec = N % 8 == 0 && !misaligned(y, 16) && !misaligned(add, 16) && !misaligned(out, 16);
    const int64_t per_block = kCombineThreads * (vec ? 8 : 1);
    const int64_t blocks_y = (N + per_block - 1) / per_block;
    if (blocks_y > 65535) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "N=%lld is too large", (long long)N);
    const dim3 grid((unsigned)T, (unsigned)blocks_y);
    auto kernel = add_f32 ? (vec ? combine_experts_kernel<8, true> : combine_experts_kernel<1, true>)
                          : (vec ? combine_experts_kernel<8, false> : combine_experts_kernel<1, false>);
    return launch(kernel, grid, kCombineThreads, 0, s, dim3(1), knobs().pdl, p);
}

int gi8_combine_experts(const void* y, const float* weights, const int32_t* places, const void* add, void* out, int64_t T, int64_t top_k,
                        int64_t rows, int64_t N, void* stream)
{
    return combine_experts(y, weights, places, add, false, out, T, top_k, rows, N, stream);
}

int gi8_combine_experts_add_f32(const void* y, const float* weights, const int32_t* places, const float* add, void* out, int64_t T, int64_t top_k,
                                int64_t rows, int64_t N, void* stream)
{
    return combine_experts(y, weights, places, add, true, out, T, top_k, rows, N, stream);
}

}  // extern "C"

// ---------------------------------------------------------------------------------------------------
// The whole layer.  Its intermediates lie one behind the other in the caller's scratch.
// ---------------------------------------------------------------------------------------------------
namespace {

struct ExpertsScratch {
    int64_t weights, experts, offsets, slots, places, counts, x_q, x_scale, h, h_q, h_scale, y, bytes;
};

ExpertsScratch experts_scratch(int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k)
{
    ExpertsScratch s{};
    const int64_t S = T * top_k;
    auto take = [&](int64_t bytes) {
        const int64_t at = s.bytes;
        s.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    s.weights = take(4 * S), s.experts = take(4 * S), s.offsets = take(4 * (E + 1)), s.slots = take(4 * S), s.places = take(4 * S);
    s.counts = take(gi8_group_by_expert_workspace_bytes(S, E));
    s.x_q = take(T * H), s.x_scale = take(4 * T);
    s.h = take(2 * S * I), s.h_q = take(S * I), s.h_scale = take(4 * S);
    s.y = take(2 * S * H);
    return s;
}

}  // namespace

extern "C" {

int64_t gi8_experts_scratch_bytes(int64_t T, int64_t H, int64_t I, int64_t E, int64_t top_k)
{
    // (what gi8_experts refuses needs none; within its limits nothing here passes 2^44)
    if (T < 0 || H < 1 || I < 1 || E < 1 || top_k < 1 || top_k > kRouteMaxTopK || T > kGroupMaxPairs / top_k || H >= kMaxK || I >= kMaxK || E > kExpertsMaxExperts) return 0;
    return experts_scratch(T, H, I, E, top_k).bytes;
}

static int experts_layer(const void* x, int x_dtype, const void* logits, int logits_dtype, const float* bias, const int8_t* gate_up,
                         const float* gate_up_scale, const int8_t* down, const float* down_scale, const void* add, bool add_f32, void* out, void* scratch,
                         int64_t scratch_bytes, int64_t T, int64_t H, int64_t I, int64_t E_router, int64_t E, int64_t first, int64_t top_k, int sigmoid,
                         int64_t groups, int64_t top_groups, int group_top2, int renormalize, float scale, void* stream)
{
    // What any step refuses is refused before the first launch: an empty batch goes through the checks of the router, and the limits of
    // the others are looked at here.
    if (int rc = gi8_route_experts(logits, logits_dtype, bias, nullptr, nullptr, 0, E_router, top_k, sigmoid, groups, top_groups, group_top2, renormalize,
                                   scale, stream))
        return rc;
    if (T < 0 || T > INT32_MAX || T * top_k > kGroupMaxPairs) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "T=%lld with top_k=%lld is out of range", (long long)T, (long long)top_k);
    if (E < 1 || E > E_router || first < 0 || first > E_router - E)
        return fail(GI8_ERR_INVALID_ARGUMENT, "%lld experts from %lld on of a router over %lld", (long long)E, (long long)first, (long long)E_router);
    if (H < 1 || I < 1 || H % 16 || I % 16) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "hidden size %lld and inner size %lld must be positive multiples of 16", (long long)H, (long long)I);
    if (H >= kMaxK || I >= kMaxK) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "hidden and inner size must be below %lld", (long long)kMaxK);
    if (E * 2 * I > INT32_MAX - 256 || E * H > INT32_MAX - 256) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "experts times channels must be below 2^31 - 256");
    if (x_dtype != 0 && x_dtype != 1) return fail(GI8_ERR_INVALID_ARGUMENT, "x_dtype must be 0 (fp32) or 1 (bf16)");
    if (T == 0) return GI8_OK;
    if (!x || !logits || !gate_up || !gate_up_scale || !down || !down_scale || !out || !scratch) return fail(GI8_ERR_INVALID_ARGUMENT, "null pointer");
    if (misaligned(x, 16) || misaligned(gate_up, 16) || misaligned(down, 16) || misaligned(scratch, 256) || misaligned(gate_up_scale, 4) || misaligned(down_scale, 4) ||
        misaligned(logits, logits_dtype == 0 ? 4 : 2) || misaligned(bias, 4) || misaligned(add, add_f32 ? 4 : 2) || misaligned(out, 2))
        return fail(GI8_ERR_MISALIGNED, "x and weights must be 16-byte aligned, scratch 256-byte aligned, the rest to its elements");
    const ExpertsScratch m = experts_scratch(T, H, I, E, top_k);
    if (scratch_bytes < m.bytes) return fail(GI8_ERR_WORKSPACE, "the layer needs %lld bytes of scratch, got %lld", (long long)m.bytes, (long long)scratch_bytes);
    uint8_t* b = static_cast<uint8_t*>(scratch);
    auto f32 = [&](int64_t at) { return reinterpret_cast<float*>(b + at); };
    auto i32 = [&](int64_t at) { return reinterpret_cast<int32_t*>(b + at); };
    auto i8 = [&](int64_t at) { return reinterpret_cast<int8_t*>(b + at); };
    const int64_t S = T * top_k;
    if (int rc = gi8_route_experts(logits, logits_dtype, bias, f32(m.weights), i32(m.experts), T, E_router, top_k, sigmoid, groups, top_groups, group_top2, renormalize,
                                   scale, stream))
        return rc;
    if (int rc = gi8_group_by_expert(i32(m.experts), S, E, first, i32(m.offsets), i32(m.slots), i32(m.places), b + m.counts, m.x_q - m.counts, stream)) return rc;
    if (int rc = gi8_quantize_token(x, x_dtype, i8(m.x_q), f32(m.x_scale), T, H, stream)) return rc;
    if (int rc = matmul_experts(i8(m.x_q), gate_up, f32(m.x_scale), gate_up_scale, i32(m.offsets), i32(m.slots), top_k, b + m.h, S, T, E, I, H, 1, stream, true)) return rc;
    if (int rc = gi8_quantize_token(b + m.h, 1, i8(m.h_q), f32(m.h_scale), S, I, stream)) return rc;
    if (int rc = matmul_experts(i8(m.h_q), down, f32(m.h_scale), down_scale, i32(m.offsets), nullptr, 1, b + m.y, S, S, E, H, I, 0, stream, true)) return rc;
    return combine_experts(b + m.y, f32(m.weights), i32(m.places), add, add_f32, out, T, top_k, S, H, stream);
}

int gi8_experts(const void* x, int x_dtype, const void* logits, int logits_dtype, const float* bias, const int8_t* gate_up,
                const float* gate_up_scale, const int8_t* down, const float* down_scale, const void* add, void* out, void* scratch,
                int64_t scratch_bytes, int64_t T, int64_t H, int64_t I, int64_t E_router, int64_t E, int64_t first, int64_t top_k, int sigmoid,
                int64_t groups, int64_t top_groups, int group_top2, int renormalize, float scale, void* stream)
{
    return experts_layer(x, x_dtype, logits, logits_dtype, bias, gate_up, gate_up_scale, down, down_scale, add, false, out, scratch, scratch_bytes, T, H, I, E_router, E, first,
                         top_k, sigmoid, groups, top_groups, group_top2, renormalize, scale, stream);
}

int gi8_experts_add_f32(const void* x, int x_dtype, const void* logits, int logits_dtype, const float* bias, const int8_t* gate_up,
                        const float* gate_up_scale, const int8_t* down, const float* down_scale, const float* add, void* out, void* scratch,
                        int64_t scratch_bytes, int64_t T, int64_t H, int64_t I, int64_t E_router, int64_t E, int64_t first, int64_t top_k, int sigmoid,
                        int64_t groups, int64_t top_groups, int group_top2, int renormalize, float scale, void* stream)
{
    return experts_layer(x, x_dtype, logits, logits_dtype, bias, gate_up, gate_up_scale, down, down_scale, add, true, out, scratch, scratch_bytes, T, H, I, E_router, E, first,
                         top_k, sigmoid, groups, top_groups, group_top2, renormalize, scale, stream);
}

}  // extern "C"
