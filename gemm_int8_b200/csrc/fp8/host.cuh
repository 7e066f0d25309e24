// C ABI of the product in 8-bit floating point and its layer: argument checks, the choice of a tile, launches.  Included at the end of api.cu,
// behind ffn/host.cuh, whose helpers it uses.
#pragma once

#include "k_fp8_gemm.cuh"

namespace {

// Tile forms and what a wave of them costs per K block, in ns (back to back; of one full wave and of many, which run at lower clocks: two-CTA 0.46 - 0.51 us, 128 x 256
// 0.44 - 0.53, 128 x 128 0.27 - 0.31, 128 x 64 0.23 - 0.26).
constexpr TileForm kFp8Forms[] = {{256, true, 480.0, 0, 0}, {256, false, 495.0, 0, 0}, {128, false, 300.0, 0, 0}, {64, false, 245.0, 0, 0}};
// What a K block takes where K is not a multiple of 32, so that rows begin inside a 32-byte sector, over what it takes where it is: for the forms in turn 0.96 - 1.06,
// 1.25 - 1.49, 1.31 - 1.52 and 1.18 - 1.38 (512 and 1024 x 4736, K = 2064, 4112, 4240, 6992 and 14352 next to the multiple of 128 below; 1024 x 4736 x 4112, us: 33.3 / 30.8,
// 40.8 / 30.2, 31.3 / 20.5, 43.0 / 33.4).  (Without this rule 1024 x 5003 x 6992 took 128 columns and 73 us, not the pair's 53.)
constexpr double kFp8OddRows[] = {1.06, 1.42, 1.47, 1.31};

struct Fp8Choice {
    int bn;
    bool pair;
    int splits;  // CTAs that share a tile's K blocks
};

// ns that a split costs beside its K blocks: two barriers of the cluster and the sums that its CTAs send each other (rows: of the tile that are stored).  Fitted to
// 32 to 256 tokens x 1024 to 8192 columns, K = 4096 to 28672, us without / with two / with four CTAs a tile: 64 x 4096 x 14336 28.7 / 19.0 (64-wide) and 17.0 (128-wide, four),
// 64 x 4096 x 4096 11.3 / 10.0 / 10.4, 40 x 2048 x 8192 18.0 / 13.3 / 11.7, 256 x 4096 x 14336 29.8 / 23.6 / 24.4, 1024 x 1024 x 8192 19.0 / 16.3 / 17.8, 100 x 1001 x 6992
// 22.0 / 16.4 / 14.9; not 300 x 300 x 1024 6.3 / 7.2, 200 x 640 x 2048 7.3 / 8.0.
double fp8_split_fixed(int bn, int splits, int64_t rows)
{
    const double part = static_cast<double>(std::min<int64_t>(4, (rows + 31) / 32)) / 4.0;
    if (bn == 64) return 2000.0 + 1000.0 * part;
    if (bn == 128) return splits == 2 ? 2500.0 + 1600.0 * part : 3900.0 + 2400.0 * part;
    return splits == 2 ? 3500.0 + 2800.0 * part : 5000.0 + 3600.0 * part;
}

// K blocks of each CTA of a split tile: a multiple of four, so that 16-byte copies of the row scales stay aligned.
int fp8_kb_per_split(int64_t kb, int splits) { return static_cast<int>((kb + 4 * splits - 1) / (4 * splits)) * 4; }

// CTAs that share a tile's K blocks in the kernel for few tokens: as many as one CTA an SM leaves room for, with eight K blocks each at least (us with 1 / 2 / 4 / 8: 16 x
// 4096 x 4096 8.6 / 7.9 / 8.0 / 12.7, 16 x 2048 x 8192 13.6 / 9.7 / 8.1 / 9.2, 1 x 1024 x 4096 8.0 / 6.3 / 5.8 / 5.6, 16 x 8192 x 8192, which has 128 CTAs, 15.1 / 20.9;
// 1 x 4096 x 1024 5.4 / 5.5).  Two CTAs an SM would fit, which long sums can use: 16 x 4096 x 14336 21.9 / 15.0 / 14.1 / 19.8, where the rule takes two.
int fp8_smallm_splits(int64_t N, int64_t K, int sms)
{
    const int64_t ctas = (N + kBwSmallTileN - 1) / kBwSmallTileN, kb = (K + kBK - 1) / kBK;
    int splits = 1;
    while (splits < 8 && ctas * splits * 2 <= sms && kb >= 8 * 2 * splits) splits *= 2;
    return splits;
}

// The form whose waves take the least time; grids that leave SMs idle are also weighed with every tile's K blocks split over the CTAs of a cluster.
// (quads: clusters of four that run at once, 33 of the 37 that 148 SMs have room for, as a cluster lies in one group of SMs: 777 x 640 x 28672 in 35 of them ran as two
// waves, 44.6 us, and takes 32.9 in pairs.)
Fp8Choice choose_fp8(int64_t M, int64_t N, int64_t K, int sms, int quads)
{
    Fp8Choice best{};
    double best_cost = 1e300;
    const int64_t kb = (K + kBK - 1) / kBK;
    for (size_t i = 0; i < sizeof(kFp8Forms) / sizeof(kFp8Forms[0]); ++i) {
        const TileForm& f = kFp8Forms[i];
        const double ns = f.kblock_cycles * (K % 32 ? kFp8OddRows[i] : 1.0);
        const int tile_m = f.pair ? 2 * kBM : kBM;
        const int64_t tiles = ((M + tile_m - 1) / tile_m) * ((N + f.bn - 1) / f.bn);
        const int64_t slots = f.pair ? sms / 2 : sms;
        const double cost = static_cast<double>((tiles + slots - 1) / slots) * ns * kb;
        if (cost < best_cost) best_cost = cost, best = {f.bn, f.pair, 1};
        if (f.pair) continue;
        for (int splits = 2; splits <= std::min(4, f.bn / 32) && tiles <= (splits == 2 ? sms / 2 : quads); splits *= 2) {
            const int each = fp8_kb_per_split(kb, splits);
            if (each * (splits - 1) >= kb) break;  // (no CTA without K blocks)
            const double split = each * ns + fp8_split_fixed(f.bn, splits, M);
            if (split < best_cost) best_cost = split, best = {f.bn, false, splits};
        }
    }
    return best;
}

// (the split kernels take an SM each; asked once per device)
int resident_quads(DeviceState* st, int* out)
{
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        *out = st->quads;
    }
    if (*out) return GI8_OK;
    constexpr size_t smem = fp8_smem_bytes(256, 4, false);
    auto kernel = fp8_gemm_kernel<256, 4, false, Fp8Bias::kNone, true>;
    if (int rc = ensure_smem(st, 75, kernel, smem)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(1, 4), cfg.blockDim = dim3(kBlockwiseThreads), cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1, attr.val.clusterDim.y = 4, attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    GI8_CUDA(cudaOccupancyMaxActiveClusters(out, kernel, &cfg));
    *out = std::max(*out, 1);
    std::lock_guard<std::mutex> lock(g_mutex);
    st->quads = *out;
    return GI8_OK;
}

template <int BN, int STAGES, bool PAIR, Fp8Bias BIAS, bool SPLITK = false>
int launch_fp8(DeviceState* st, int slot, const int8_t* x, const int8_t* y, Fp8GemmParams p, cudaStream_t s)
{
    constexpr size_t smem = fp8_smem_bytes(BN, STAGES, PAIR);
    static_assert(smem <= 227 * 1024 - 512, "shared memory per CTA");
    auto kernel = fp8_gemm_kernel<BN, STAGES, PAIR, BIAS, SPLITK>;
    if (int rc = ensure_smem(st, slot, kernel, smem)) return rc;
    CUtensorMap mx, my, mo{};
    // No more rows than there are, in whole groups of eight (the swizzle's): boxes of 128 rows over x of less than 128 KB were slow, 17 x 14336 x 4096 17.1 us for 11.3
    // (x 32 rows, which are 128 KB: 11.6 and 11.3), 24 x 4096 x 4096 11.7 for 9.4.
    p.box_rows = PAIR ? kBM : std::min(kBM, (p.M + 7) / 8 * 8);
    if (int rc = make_operand_map(&mx, x, p.M, p.K, p.box_rows)) return rc;
    if (int rc = make_operand_map(&my, y, p.N, p.K, PAIR ? BN / 4 : BN)) return rc;
    if (p.tma_store)
        if (int rc = make_output_map(&mo, p.out, p.M, p.N, p.ldo, kFp8StoreCols)) return rc;
    constexpr int kTileM = PAIR ? 2 * kBM : kBM;
    p.tiles_m = (p.M + kTileM - 1) / kTileM, p.tiles_n = (p.N + BN - 1) / BN;
    p.group_m = pick_group_m(p.K);
    if (PAIR) p.group_m = std::max(1, p.group_m / 2);
    const int64_t tiles = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    const int slots = PAIR ? st->sm_count / 2 : st->sm_count;
    const int grid = static_cast<int>(std::min<int64_t>(tiles, slots)) * (PAIR ? 2 : 1);
    const int64_t ctas = tiles * (SPLITK ? p.splits : 1);
    p.release_late = !PAIR && !(p.after_quant && BN < 256) && (ctas <= st->sm_count || p.K % 32 != 0) && release_late(ctas, st->sm_count);
    if constexpr (SPLITK) return launch(kernel, dim3(static_cast<unsigned>(tiles), p.splits), kBlockwiseThreads, smem, s, dim3(1, p.splits), knobs().pdl, mx, my, mo, p);
    return launch(kernel, dim3(grid), kBlockwiseThreads, smem, s, dim3(PAIR ? 2 : 1), knobs().pdl, mx, my, mo, p);
}

template <Fp8Bias BIAS>
int launch_fp8(DeviceState* st, Fp8Choice c, const int8_t* x, const int8_t* y, const Fp8GemmParams& p, cudaStream_t s)
{
    constexpr int slot = BIAS == Fp8Bias::kBf16 ? 64 : BIAS == Fp8Bias::kNone ? 71 : 80;
    if (c.splits > 1) {
        Fp8GemmParams q = p;
        q.splits = c.splits, q.kb_per_split = fp8_kb_per_split((p.K + kBK - 1) / kBK, c.splits);
        if (c.bn == 256) return launch_fp8<256, 4, false, BIAS, true>(st, slot + 4, x, y, q, s);
        if (c.bn == 128) return launch_fp8<128, 6, false, BIAS, true>(st, slot + 5, x, y, q, s);
        return launch_fp8<64, 8, false, BIAS, true>(st, slot + 6, x, y, q, s);
    }
    if (c.pair) return launch_fp8<256, 6, true, BIAS>(st, slot, x, y, p, s);
    if (c.bn == 256) return launch_fp8<256, 4, false, BIAS>(st, slot + 1, x, y, p, s);
    if (c.bn == 128) return launch_fp8<128, 6, false, BIAS>(st, slot + 2, x, y, p, s);
    return launch_fp8<64, 8, false, BIAS>(st, slot + 3, x, y, p, s);
}

// (bias bf16 or fp32, or null; after_quant: see scaled_impl)
int fp8_matmul(const int8_t* x, const int8_t* y, const float* sa, int64_t ld_sa, const float* sw, int64_t ld_sw, void* out, int64_t M, int64_t N, int64_t K,
               void* stream, const void* bias, bool bias_f32, bool after_quant)
{
    if (int rc = check_common(x, y, out, M, N, K, 2)) return rc;
    if (M == 0 || N == 0) return GI8_OK;
    if (K > 0)
        if (int rc = check_block_scales(sa, ld_sa, sw, ld_sw, M, N, K)) return rc;
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (K == 0) return zero_output(out, M * N * 2, s);
    after_quant = after_quant && knobs().pdl;
    const int forced = g_forced_variant;
    if (forced == VAR_AUTO && use_blockwise_smallm(M, N, K)) {
        BlockwiseSmallMParams q{};
        q.out = static_cast<uint16_t*>(out), q.sa = sa, q.sw = sw, q.bias = static_cast<const uint16_t*>(bias), q.bias_f32 = bias_f32, q.status = st->status;
        q.ldo = N, q.ld_sa = ld_sa, q.ld_sw = ld_sw, q.M = (int)M, q.N = (int)N, q.K = (int)K;
        q.after_quant = after_quant;
        q.splits = fp8_smallm_splits(N, K, st->sm_count);
        q.kb_per_split = static_cast<int>(((K + kBK - 1) / kBK + q.splits - 1) / q.splits);
        if (q.splits == 1 && blockwise_smallm_six_stages(N, K, q.after_quant, st->sm_count)) return launch_blockwise_smallm<6, E4m3>(st, 79, x, y, q, s);
        return launch_blockwise_smallm<4, E4m3>(st, 78, x, y, q, s);
    }
    Fp8GemmParams p{};
    p.out = out, p.sa = sa, p.sw = sw, p.bias = bias, p.status = st->status, p.ldo = N, p.ld_sa = ld_sa, p.ld_sw = ld_sw;
    p.M = (int)M, p.N = (int)N, p.K = (int)K;
    p.tma_store = !misaligned(out, 16) && N % 8 == 0 && knobs().tma_store;
    p.pair_ok = !misaligned(out, 4) && N % 2 == 0;
    p.bias_vec = !misaligned(bias, 16);
    p.after_quant = after_quant;
    p.scale_vec = (K + kBK - 1) / kBK % 4 == 0 && ld_sa % 4 == 0 && !misaligned(sa, 16);
    Fp8Choice c;
    switch (forced) {
        case VAR_DENSE_BN256: c = {256, false, 1}; break;
        case VAR_DENSE_BN128: c = {128, false, 1}; break;
        case VAR_DENSE_BN64: c = {64, false, 1}; break;
        case VAR_PAIR: c = {256, true, 1}; break;
        default: {
            int quads;
            if (int rc = resident_quads(st, &quads)) return rc;
            c = choose_fp8(M, N, K, st->sm_count, quads);
        }
    }
    if (!bias) return launch_fp8<Fp8Bias::kNone>(st, c, x, y, p, s);
    return bias_f32 ? launch_fp8<Fp8Bias::kF32>(st, c, x, y, p, s) : launch_fp8<Fp8Bias::kBf16>(st, c, x, y, p, s);
}

int fp8_linear(const void* x, int x_dtype, const void* w, const float* w_scale, int64_t ld_sw, const void* bias, bool bias_f32, void* xq, float* xs, void* out,
               int64_t M, int64_t N, int64_t K, void* stream)
{
    // Everything that the quantiser or the product refuses is refused before the quantiser is launched (as in gi8_linear).
    if (int rc = check_common(xq, w, out, M, N, K, 2)) return rc;
    if (int rc = check_quant(x, x_dtype, static_cast<const int8_t*>(xq), xs, M, K)) return rc;
    if (misaligned(bias, bias_f32 ? 4 : 2)) return fail(GI8_ERR_MISALIGNED, "bias must be aligned to its type");
    if (M == 0 || N == 0) return GI8_OK;
    if (K == 0 && bias) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "K must be positive for a product with a bias");
    const int64_t ld_xs = (K + kBK - 1) / kBK;
    if (K > 0)
        if (int rc = check_block_scales(xs, ld_xs, w_scale, ld_sw, M, N, K)) return rc;
    if (int rc = gi8_fp8_quantize_token_block(x, x_dtype, xq, xs, M, K, stream)) return rc;
    return fp8_matmul(static_cast<const int8_t*>(xq), static_cast<const int8_t*>(w), xs, ld_xs, w_scale, ld_sw, out, M, N, K, stream,
                      bias, bias_f32, K > 0);
}

}  // namespace

extern "C" {

int gi8_fp8_quantize_token_block(const void* in, int in_dtype, void* q, float* scales, int64_t M, int64_t K, void* stream)
{
    if (int rc = check_quant(in, in_dtype, static_cast<const int8_t*>(q), scales, M, K)) return rc;
    if (K % 8) return fail(GI8_ERR_UNSUPPORTED_SHAPE, "K=%lld must be a multiple of 8", (long long)K);
    if (M == 0 || K == 0) return GI8_OK;
    DeviceState* st;
    if (int rc = get_device_state(&st)) return rc;
    ActParams p{in, static_cast<uint8_t*>(q), scales, M, static_cast<int>(K), static_cast<int>((K + 127) / 128)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return in_dtype == 0 ? launch_act_block<float, false, Out8::kE4m3>(p, s) : launch_act_block<__nv_bfloat16, false, Out8::kE4m3>(p, s);
}

int gi8_fp8_matmul_blockwise(const void* x, const void* y, const float* sa, int64_t ld_sa, const float* sw, int64_t ld_sw, void* out, int64_t M, int64_t N,
                             int64_t K, void* stream)
{
    return fp8_matmul(static_cast<const int8_t*>(x), static_cast<const int8_t*>(y), sa, ld_sa, sw, ld_sw, out, M, N, K, stream, nullptr, false, false);
}

int gi8_fp8_linear(const void* x, int x_dtype, const void* w, const float* w_scale, int64_t ld_sw, const void* bias, void* xq, float* xs, void* out,
                   int64_t M, int64_t N, int64_t K, void* stream)
{
    return fp8_linear(x, x_dtype, w, w_scale, ld_sw, bias, false, xq, xs, out, M, N, K, stream);
}

int gi8_fp8_linear_bias_f32(const void* x, int x_dtype, const void* w, const float* w_scale, int64_t ld_sw, const float* bias, void* xq, float* xs,
                            void* out, int64_t M, int64_t N, int64_t K, void* stream)
{
    return fp8_linear(x, x_dtype, w, w_scale, ld_sw, bias, true, xq, xs, out, M, N, K, stream);
}

}  // extern "C"
